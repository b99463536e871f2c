// CPython extension m2_amd._causal_calls: the host side of causal_conv, selective_scan, their steps, and group_norm (m2_amd/causal.py, m2_amd/ops.py): checks, output
// tensors, the call into libm2_amd.so and the nodes of the graph.  A token's step is a few microseconds on the GPU, less than the same in Python would take.
#include <c10/hip/HIPGraphsC10Utils.h>

#include "torch_calls.h"

namespace {

decltype(&m2_causal_conv_fwd) conv_fwd;
decltype(&m2_causal_conv_bwd_workspace_bytes) conv_bwd_workspace_bytes;
decltype(&m2_causal_conv_bwd) conv_bwd;
decltype(&m2_causal_conv_step) conv_step;
decltype(&m2_selective_scan_span) scan_span;
decltype(&m2_selective_scan_fwd) scan_fwd;
decltype(&m2_selective_scan_bwd_workspace_bytes) scan_bwd_workspace_bytes;
decltype(&m2_selective_scan_bwd) scan_bwd;
decltype(&m2_selective_scan_step) scan_step;
decltype(&m2_group_norm_workspace_bytes) norm_workspace_bytes;
decltype(&m2_group_norm_fwd) norm_fwd;
decltype(&m2_group_norm_bwd) norm_bwd;

void bind(const std::vector<uintptr_t>& a) {
  TORCH_CHECK(a.size() == 13, "thirteen addresses");
  set(last_error, a[0]);
  set(conv_fwd, a[1]);
  set(conv_bwd_workspace_bytes, a[2]);
  set(conv_bwd, a[3]);
  set(conv_step, a[4]);
  set(scan_span, a[5]);
  set(scan_fwd, a[6]);
  set(scan_bwd_workspace_bytes, a[7]);
  set(scan_bwd, a[8]);
  set(scan_step, a[9]);
  set(norm_workspace_bytes, a[10]);
  set(norm_fwd, a[11]);
  set(norm_bwd, a[12]);
}

constexpr int64_t kMost = 1 << 30;      // of a size that goes through the C entry points as int

// t (undefined: not given) on `like`'s device, of a type and sizes.
void expect(const char* name, const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  if (!t.defined()) return;
  TORCH_CHECK(t.device() == like.device(), name, ": must live on ", like.device(), ", got ", t.device());
  TORCH_CHECK_TYPE(t.layout() == at::kStrided && t.scalar_type() == type, name, ": expected ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, ": expected ", sizes, ", got ", t.sizes());
}
void positive(const char* name, const Tensor& t, int64_t first) {
  for (int64_t i = first; i < t.dim(); ++i) TORCH_CHECK_VALUE(t.size(i) > 0 && t.size(i) <= kMost, name, ": sizes must be positive and at most 2^30, got ", t.sizes());
  TORCH_CHECK_VALUE(first == 0 || t.size(0) <= kMost, name, ": sizes must be at most 2^30, got ", t.sizes());
}

// t with its values one behind the other along the last `last` dimensions, the leading ones any distance apart.
Tensor rows(const Tensor& t, int64_t last = 1) {
  if (!t.defined()) return t;
  if (t.is_neg()) return t.resolve_neg().contiguous();
  int64_t expected = 1;
  for (int64_t i = t.dim() - 1; i >= t.dim() - last; --i) {
    if (t.size(i) != 1 && t.stride(i) != expected) return t.contiguous();
    expected *= t.size(i);
  }
  return t;
}
// t (B, L, ...) of what the scan's kernels address in 32 bits from a position on: rows below 2^24 values apart.
Tensor near_rows(const Tensor& t) { return t.defined() && t.size(1) > 1 && t.stride(1) >= 1 << 24 ? t.contiguous() : t; }
int64_t row_of(const Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }
const float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
float* floats_out(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const long long* lengths_of(const Tensor& t) { return t.defined() ? reinterpret_cast<const long long*>(t.data_ptr<int64_t>()) : nullptr; }
Tensor scratch(size_t bytes, const Tensor& like) { return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor(); }

// The bytes that t's values lie in.
std::pair<uintptr_t, uintptr_t> extent(const Tensor& t) {
  int64_t most = 0;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 0) return {0, 0};
    most += (t.size(i) - 1) * t.stride(i);
  }
  const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {at, at + (most + 1) * t.element_size()};
}
bool apart(const Tensor& a, const Tensor& b) {
  if (!a.defined() || !b.defined()) return true;
  const auto [a0, a1] = extent(a);
  const auto [b0, b1] = extent(b);
  return a1 <= b0 || b1 <= a0;
}

// A step's state and where the next one goes: in place, or another tensor that shares no memory with what the step reads.
Tensor next_state(const Tensor& state, const optional<Tensor>& out_state, std::initializer_list<Tensor> read) {
  const Tensor next = out_state ? *out_state : state;
  const bool in_place = next.data_ptr() == state.data_ptr();
  if (out_state) expect("out_state", next, state, state.scalar_type(), state.sizes());
  TORCH_CHECK_VALUE(state.is_contiguous() && !state.is_neg() && next.is_contiguous() && !next.is_neg(), "state and out_state must be contiguous");
  TORCH_CHECK_VALUE(in_place || apart(next, state), "out_state: shares memory with state");
  for (const Tensor& t : read) TORCH_CHECK_VALUE(apart(next, t), "the state that is written shares memory with an input");
  return next;
}

// A backward pass inside a stream capture goes to the streams on which its leaves' accumulators were made: one that an eager graph of another stream keeps alive
// would take the capture there, which ends the process.  Refused while the forward can still be.
void refuse_other_graphs(std::initializer_list<Tensor> inputs) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    const auto made = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!made) continue;
    const optional<c10::Stream> stream = made->stream();
    TORCH_CHECK(!stream || *stream == c10::hip::getCurrentHIPStream(t.device().index()).unwrap(),
                "stream capture: a graph made on another stream still holds an input that asks for gradients; let go of its outputs first, or detach the input");
  }
}

bool asks(std::initializer_list<Tensor> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : inputs)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// What is asked of the gradients of gradients has to fail.
variable_list without_second(const char* name, variable_list g) {
  if (!at::GradMode::is_enabled()) return g;
  for (Tensor& t : g) {
    if (!t.defined()) continue;
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative", 1);
    t.set_requires_grad(true);
    t = (*node)({t})[0];
  }
  return g;
}

// A node with saved inputs.  Hooks on saved tensors (torch.autograd.graph.saved_tensors_hooks) may hand out others than were saved: types and sizes are checked again.
struct CausalNode : torch::autograd::Node {
  std::vector<SavedVariable> saved;
  struct Kind {
    bool defined;
    at::ScalarType type;
    std::vector<int64_t> sizes;
  };
  std::vector<Kind> kinds;
  bool released = false;

  void save(std::initializer_list<Tensor> tensors) {
    for (const Tensor& t : tensors) {
      saved.emplace_back(t, false);
      kinds.push_back(t.defined() ? Kind{true, t.scalar_type(), t.sizes().vec()} : Kind{false, at::kFloat, {}});
    }
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& v : saved) v.reset_data();
    released = true;
  }
  std::vector<Tensor> unpack() {
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    std::vector<Tensor> t;
    for (size_t i = 0; i < saved.size(); ++i) {
      t.push_back(saved[i].unpack());
      TORCH_CHECK(t[i].defined() == kinds[i].defined && (!t[i].defined() || (t[i].is_cuda() && t[i].device() == t[0].device() && t[i].layout() == at::kStrided &&
                  t[i].scalar_type() == kinds[i].type && t[i].sizes() == at::IntArrayRef(kinds[i].sizes))), name(), ": a saved tensor came back as another one");
    }
    return t;
  }
};
template <typename N>
std::shared_ptr<N> new_node(std::initializer_list<Tensor> inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  for (const Tensor& t : inputs) edges.push_back(t.defined() && t.requires_grad() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
  node->set_next_edges(std::move(edges));
  return node;
}
Tensor given(const Tensor& g, const Tensor& like) { return g.defined() ? rows(g) : at::zeros({like.size(-1)}, like.options().requires_grad(false)).expand(like.sizes()); }

// ---- causal convolution ---------------------------------------------------------------------------------------------------------------------------------------

struct Conv {
  Tensor x, w, bias, state, lengths;      // x (B, L, C) or, a step's, (B, C)
  int type;
  int64_t B, L, C, K;
  bool silu;
};
Conv conv_of(const Tensor& x, const Tensor& w, const Tensor& bias, bool silu, const Tensor& state, const Tensor& lengths, bool step) {
  Conv c{x, w, bias, state, lengths};
  c.type = type_of("x", x);
  TORCH_CHECK_VALUE(x.dim() == (step ? 2 : 3), "x: expected ", step ? "(B, C)" : "(B, L, C)", ", got ", x.sizes());
  positive("x", x, 1);
  c.B = x.size(0), c.L = step ? 1 : x.size(1), c.C = x.size(-1);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == c.C && w.size(1) >= 1 && w.size(1) <= 8, "weight: expected (", c.C, ", 1 to 8 taps), got ", w.sizes());
  c.K = w.size(1);
  expect("weight", w, x, at::kFloat, {c.C, c.K});
  expect("bias", bias, x, at::kFloat, {c.C});
  expect("state", state, x, x.scalar_type(), {c.B, c.K - 1, c.C});
  expect("lengths", lengths, x, at::kLong, {c.B});
  c.silu = silu;
  return c;
}

// y and, if wanted, the state behind the last position.
std::pair<Tensor, Tensor> conv(const Conv& c, bool want_state) {
  const c10::DeviceGuard guard(c.x.device());
  const auto options = c.x.options().requires_grad(false);
  Tensor y = at::empty({c.B, c.L, c.C}, options), last = want_state ? at::empty({c.B, c.K - 1, c.C}, options) : Tensor();
  if (c.B == 0) return {y, last};
  const Tensor x = rows(c.x), w = dense(c.w), bias = dense(c.bias), state = dense(c.state), lengths = dense(c.lengths);
  check(conv_fwd(x.data_ptr(), x.stride(0), x.stride(1), floats(w), floats(bias), pointer(state), lengths_of(lengths), y.data_ptr(), pointer(last), c.B, c.L, c.C, c.K, c.silu, c.type,
                 current_stream()));
  return {y, last};
}

struct CausalConvBackward : CausalNode {
  int type = 0;
  bool silu = false, states = false;

  std::string name() const override { return "CausalConvBackward"; }

  variable_list apply(variable_list&& g) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const std::vector<Tensor> in = unpack();
    if (!g[0].defined() && !g[1].defined()) return variable_list(4);
    variable_list out(4);      // x, weight, bias, state
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(in[0].device());
      const Tensor x = rows(in[0]), w = dense(in[1]), bias = dense(in[2]), state = dense(in[3]), lengths = dense(in[4]), gy = given(g[0], x), glast = dense(g[1]);
      for (int i = 0; i < 4; ++i)
        if (task_should_compute_output(i)) out[i] = at::empty(in[i].sizes(), in[i].options().requires_grad(false));
      const int64_t B = x.size(0), L = x.size(1), C = x.size(2), K = w.size(1);
      if (B == 0) {
        for (Tensor& t : out)
          if (t.defined()) t.zero_();
      } else {
        const Tensor room = out[1].defined() || out[2].defined() ? scratch(conv_bwd_workspace_bytes(B, L, C, K, type), x) : Tensor();
        check(conv_bwd(x.data_ptr(), x.stride(0), x.stride(1), floats(w), floats(bias), pointer(state), lengths_of(lengths), gy.data_ptr(), gy.stride(0), gy.stride(1), pointer(glast),
                       pointer(out[0]), floats_out(out[1]), floats_out(out[2]), K > 1 ? pointer(out[3]) : nullptr, pointer(room), B, L, C, K, silu, type, current_stream()));
      }
    }
    return without_second("causal_conv", std::move(out));
  }
};

std::pair<Tensor, Tensor> causal_conv(const Tensor& x, const Tensor& w, const Tensor& bias, bool silu, const Tensor& state, const Tensor& lengths, bool want_state) {
  const Conv c = conv_of(x, w, bias, silu, state, lengths, false);
  if (!asks({x, w, bias, state})) return conv(c, want_state);
  const c10::DeviceGuard guard(x.device());
  refuse_other_graphs({x, w, bias, state});
  const auto node = new_node<CausalConvBackward>({x, w, bias, state});
  std::pair<Tensor, Tensor> out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = conv(c, want_state);
  }
  torch::autograd::set_history(variable_list{out.first, out.second}, node);
  node->save({x, w, bias, state, lengths});
  node->type = c.type, node->silu = silu;
  return out;
}

Tensor causal_conv_step(const Tensor& x, const Tensor& state, const Tensor& w, const Tensor& bias, bool silu, const optional<Tensor>& out_state) {
  const Conv c = conv_of(x, w, bias, silu, state, Tensor(), true);
  const Tensor next = next_state(state, out_state, {x, w, bias});
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty({c.B, c.C}, x.options().requires_grad(false));
  if (c.B == 0) return y;
  const Tensor in = rows(x), taps = dense(w), offsets = dense(bias);
  next.unsafeGetTensorImpl()->bump_version();
  check(conv_step(in.data_ptr(), in.stride(0), state.data_ptr(), floats(taps), floats(offsets), y.data_ptr(), next.data_ptr(), c.B, c.C, c.K, silu, c.type, current_stream()));
  return y;
}

// ---- selective scan -------------------------------------------------------------------------------------------------------------------------------------------

enum { X, DT, A_, B_, C_, D_, Z, DT_BIAS, STATE, INPUTS, LENGTHS = INPUTS, SAVED, SCAN_SAVED };

struct Scan {
  std::vector<Tensor> in;      // in that order, up to LENGTHS
  int type;
  int64_t batch, L, D, G, N;
  bool softplus, step;
};
Scan scan_of(std::vector<Tensor> in, bool softplus, bool step) {
  Scan s;
  const Tensor &x = in[X], &A = in[A_];
  s.type = type_of("x", x);
  TORCH_CHECK_VALUE(x.dim() == (step ? 2 : 3), "x: expected ", step ? "(B, D)" : "(B, L, D)", ", got ", x.sizes());
  positive("x", x, 1);
  s.batch = x.size(0), s.L = step ? 1 : x.size(1), s.D = x.size(-1);
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == s.D && A.size(1) >= 1 && A.size(1) <= 256, "A: expected (", s.D, ", 1 to 256 states), got ", A.sizes());
  s.N = A.size(1);
  expect("A", A, x, at::kFloat, {s.D, s.N});
  expect("dt", in[DT], x, x.scalar_type(), x.sizes());
  expect("z", in[Z], x, x.scalar_type(), x.sizes());
  const int64_t lead = x.dim() - 1;
  TORCH_CHECK_VALUE(in[B_].dim() == lead + 1 || in[B_].dim() == lead + 2, "B: expected (..., groups, ", s.N, ") or (..., ", s.N, "), got ", in[B_].sizes());
  s.G = in[B_].dim() == lead + 2 ? in[B_].size(-2) : 1;
  TORCH_CHECK_VALUE(s.G >= 1 && s.D % s.G == 0, "B: ", s.G, " groups do not divide ", s.D, " channels");
  std::vector<int64_t> shared = x.sizes().slice(0, lead).vec();
  if (in[B_].dim() == lead + 2) shared.push_back(s.G);
  shared.push_back(s.N);
  expect("B", in[B_], x, x.scalar_type(), shared);
  expect("C", in[C_], x, x.scalar_type(), shared);
  expect("D", in[D_], x, at::kFloat, {s.D});
  expect("dt_bias", in[DT_BIAS], x, at::kFloat, {s.D});
  expect("state", in[STATE], x, at::kFloat, {s.batch, s.D, s.N});
  if (in.size() > LENGTHS) expect("lengths", in[LENGTHS], x, at::kLong, {s.batch});
  s.in = std::move(in);
  s.softplus = softplus, s.step = step;
  return s;
}

// What the library is given, and the tensors that hold it.
struct ScanCall {
  std::vector<Tensor> keep;
  m2_scan_inputs in{};

  explicit ScanCall(const Scan& s) {
    for (int i = 0; i < INPUTS; ++i) keep.push_back(i == X || i == DT || i == Z || i == B_ || i == C_ ? rows(s.in[i]) : dense(s.in[i]));
    keep.push_back(s.in.size() > LENGTHS ? dense(s.in[LENGTHS]) : Tensor());
    const auto place = [&](int i, const void*& p, long& batch, long& row) {
      if (!keep[i].defined()) return;
      if (!s.step) keep[i] = near_rows(keep[i]);
      p = keep[i].data_ptr(), batch = keep[i].stride(0), row = s.step ? 0 : row_of(keep[i]);
    };
    place(X, in.x, in.x_batch, in.x_row);
    place(DT, in.dt, in.dt_batch, in.dt_row);
    place(Z, in.z, in.z_batch, in.z_row);
    place(B_, in.Bm, in.b_batch, in.b_row);
    place(C_, in.Cm, in.c_batch, in.c_row);
    const bool groups = keep[B_].dim() == (s.step ? 3 : 4);
    in.b_group = groups ? keep[B_].stride(-2) : 0, in.c_group = groups ? keep[C_].stride(-2) : 0;
    in.A = floats(keep[A_]), in.D = floats(keep[D_]), in.dt_bias = floats(keep[DT_BIAS]), in.state = floats(keep[STATE]), in.lengths = lengths_of(keep[LENGTHS]);
    in.batch = s.batch, in.length = s.L, in.channels = s.D, in.groups = s.G, in.states = s.N, in.softplus = s.softplus;
  }
};

// y, the last state if wanted, and what the gradient needs of the states if that is wanted.
std::array<Tensor, 3> scan(const Scan& s, bool want_state, bool want_saved) {
  const Tensor& x = s.in[X];
  const c10::DeviceGuard guard(x.device());
  const auto options = x.options().requires_grad(false), f32 = options.dtype(at::kFloat);
  std::array<Tensor, 3> out;
  out[0] = at::empty({s.batch, s.L, s.D}, options);
  if (want_state) out[1] = at::empty({s.batch, s.D, s.N}, f32);
  if (want_saved) {
    const int64_t span = scan_span(s.N);
    out[2] = at::empty({s.batch, (s.L + span - 1) / span, s.D, s.N}, f32);
  }
  if (s.batch == 0) return out;
  const ScanCall call(s);
  check(scan_fwd(&call.in, out[0].data_ptr(), floats_out(out[1]), floats_out(out[2]), s.type, current_stream()));
  return out;
}

struct SelectiveScanBackward : CausalNode {
  bool softplus = false;

  std::string name() const override { return "SelectiveScanBackward"; }

  variable_list apply(variable_list&& g) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    std::vector<Tensor> in = unpack();
    if (!g[0].defined() && !g[1].defined()) return variable_list(INPUTS);
    variable_list out(INPUTS);
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(in[X].device());
      const Tensor kept = dense(in[SAVED]), gy = near_rows(given(g[0], in[X])), glast = dense(g[1]);
      for (int i = 0; i < INPUTS; ++i)
        if (task_should_compute_output(i)) out[i] = at::empty(in[i].sizes(), in[i].options().requires_grad(false));
      in.pop_back();
      const Scan s = scan_of(std::move(in), softplus, false);
      if (s.batch == 0) {
        for (Tensor& t : out)
          if (t.defined()) t.zero_();
      } else {
        const ScanCall call(s);
        const Tensor room = scratch(scan_bwd_workspace_bytes(s.batch, s.L, s.D, s.G, s.N), s.in[X]);
        m2_scan_gradients into{};
        into.gy = gy.data_ptr(), into.gy_batch = gy.stride(0), into.gy_row = row_of(gy), into.gstate_out = floats(glast);
        into.gx = pointer(out[X]), into.gdt = pointer(out[DT]), into.gz = pointer(out[Z]), into.gB = pointer(out[B_]), into.gC = pointer(out[C_]);
        into.gA = floats_out(out[A_]), into.gD = floats_out(out[D_]), into.gdt_bias = floats_out(out[DT_BIAS]), into.gstate = floats_out(out[STATE]);
        check(scan_bwd(&call.in, &into, floats(kept), pointer(room), s.type, current_stream()));
      }
    }
    return without_second("selective_scan", std::move(out));
  }
};

std::pair<Tensor, Tensor> selective_scan(std::vector<Tensor> in, bool softplus, bool want_state) {
  const Scan s = scan_of(std::move(in), softplus, false);
  const std::vector<Tensor>& t = s.in;
  const std::initializer_list<Tensor> inputs = {t[X], t[DT], t[A_], t[B_], t[C_], t[D_], t[Z], t[DT_BIAS], t[STATE]};
  if (!asks(inputs)) {
    auto out = scan(s, want_state, false);
    return {out[0], out[1]};
  }
  const c10::DeviceGuard guard(t[X].device());
  refuse_other_graphs(inputs);
  const auto node = new_node<SelectiveScanBackward>(inputs);
  std::array<Tensor, 3> out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = scan(s, want_state, true);
  }
  torch::autograd::set_history(variable_list{out[0], out[1]}, node);
  node->save({t[X], t[DT], t[A_], t[B_], t[C_], t[D_], t[Z], t[DT_BIAS], t[STATE], t[LENGTHS], out[2]});
  node->softplus = softplus;
  return {out[0], out[1]};
}

Tensor selective_scan_step(std::vector<Tensor> in, bool softplus, const optional<Tensor>& out_state) {
  const Scan s = scan_of(std::move(in), softplus, true);
  const std::vector<Tensor>& t = s.in;
  const Tensor next = next_state(t[STATE], out_state, {t[X], t[DT], t[A_], t[B_], t[C_], t[D_], t[Z], t[DT_BIAS]});
  const c10::DeviceGuard guard(t[X].device());
  Tensor y = at::empty({s.batch, s.D}, t[X].options().requires_grad(false));
  if (s.batch == 0) return y;
  const ScanCall call(s);
  next.unsafeGetTensorImpl()->bump_version();
  check(scan_step(&call.in, y.data_ptr(), next.data_ptr<float>(), s.type, current_stream()));
  return y;
}

// ---- group norm -----------------------------------------------------------------------------------------------------------------------------------------------

struct Norm {
  Tensor x, w, b;
  int type, act;
  int64_t N, S, C, G;
  double eps;
};
Norm norm_of(const Tensor& x, int64_t G, const Tensor& w, const Tensor& b, double eps, int act) {
  Norm n{x, w, b};
  n.type = type_of("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 2, "x: expected (N, ..., C), got ", x.sizes());
  positive("x", x, 1);
  n.N = x.size(0), n.C = x.size(-1), n.S = 1;
  for (int64_t i = 1; i < x.dim() - 1; ++i) n.S *= x.size(i);
  TORCH_CHECK_VALUE(n.S <= kMost, "x: at most 2^30 positions of a sample, got ", x.sizes());
  TORCH_CHECK_VALUE(G >= 1 && n.C % G == 0, "groups: ", G, " do not divide ", n.C, " channels");
  TORCH_CHECK_VALUE(eps >= 0, "eps: must not be negative, got ", eps);
  expect("weight", w, x, at::kFloat, {n.C});
  expect("bias", b, x, at::kFloat, {n.C});
  n.G = G, n.act = act, n.eps = eps;
  return n;
}

// x (N, ..., C) as samples of S rows of C values: where they begin, a sample and a row apart; a copy where the rows lie at more than one distance.
struct Samples {
  Tensor t;
  int64_t sample, row;
};
Samples samples(const Tensor& x) {
  Tensor t = rows(x);
  for (bool again = false;; again = true) {
    int64_t size = 1, stride = t.size(-1);
    bool one = true;
    for (int64_t i = t.dim() - 2; i >= 1; --i) {
      if (t.size(i) == 1) continue;
      if (size == 1) stride = t.stride(i);
      else one = one && t.stride(i) == size * stride;
      size *= t.size(i);
    }
    if (one || again) return {t, t.stride(0), stride};
    t = t.contiguous();
  }
}

std::pair<Tensor, Tensor> norm(const Norm& n) {
  const c10::DeviceGuard guard(n.x.device());
  const auto options = n.x.options().requires_grad(false);
  Tensor y = at::empty(n.x.sizes(), options, at::MemoryFormat::Contiguous), stats = at::empty({n.N, n.G, 2}, options.dtype(at::kFloat));
  if (n.N == 0) return {y, stats};
  const Samples x = samples(n.x);
  const Tensor w = dense(n.w), b = dense(n.b), room = scratch(norm_workspace_bytes(n.N, n.S, n.C, n.G, 0, n.type), n.x);
  check(norm_fwd(x.t.data_ptr(), x.sample, x.row, floats(w), floats(b), static_cast<float>(n.eps), y.data_ptr(), floats_out(stats), pointer(room), n.N, n.S, n.C, n.G, n.act, n.type,
                 current_stream()));
  return {y, stats};
}

struct GroupNormBackward : CausalNode {
  int act = 0;
  int64_t groups = 1;

  std::string name() const override { return "GroupNormBackward"; }

  variable_list apply(variable_list&& g) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const std::vector<Tensor> in = unpack();
    variable_list out(3);
    if (!g[0].defined()) return out;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(in[0].device());
      const Norm n = norm_of(in[0], groups, in[1], in[2], 0., act);
      for (int i = 0; i < 3; ++i)
        if (task_should_compute_output(i)) out[i] = at::empty(in[i].sizes(), in[i].options().requires_grad(false), at::MemoryFormat::Contiguous);
      if (n.N == 0) {
        for (Tensor& t : out)
          if (t.defined()) t.zero_();
      } else {
        const Samples x = samples(n.x), gy = samples(g[0]);
        const Tensor w = dense(n.w), b = dense(n.b), stats = dense(in[3]), room = scratch(norm_workspace_bytes(n.N, n.S, n.C, n.G, 1, n.type), n.x);
        check(norm_bwd(x.t.data_ptr(), x.sample, x.row, floats(w), floats(b), floats(stats), gy.t.data_ptr(), gy.sample, gy.row, pointer(out[0]), floats_out(out[1]), floats_out(out[2]),
                       pointer(room), n.N, n.S, n.C, n.G, n.act, n.type, current_stream()));
      }
    }
    return without_second("group_norm", std::move(out));
  }
};

Tensor group_norm(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps, int act) {
  const Norm n = norm_of(x, groups, w, b, eps, act);
  if (!asks({x, w, b})) return norm(n).first;
  const c10::DeviceGuard guard(x.device());
  refuse_other_graphs({x, w, b});
  const auto node = new_node<GroupNormBackward>({x, w, b});
  std::pair<Tensor, Tensor> out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = norm(n);
  }
  torch::autograd::set_history(out.first, node);
  node->save({x, w, b, out.second});
  node->act = act, node->groups = groups;
  return out.first;
}

// ---- arguments ------------------------------------------------------------------------------------------------------------------------------------------------

Tensor maybe(const char* name, PyObject* o, bool grad_ok) { return o == Py_None ? Tensor() : values(name, o, grad_ok); }

PyObject* pair_of(std::pair<Tensor, Tensor> found) {
  auto results = pybind11::reinterpret_steal<pybind11::object>(PyTuple_New(2));
  if (!results) throw python_error();
  for (int i = 0; i < 2; ++i) {
    PyObject* o = object_of(std::move(i ? found.second : found.first));
    if (!o) throw python_error();
    PyTuple_SET_ITEM(results.ptr(), i, o);
  }
  return results.release().ptr();
}

// (x, weight, bias, silu, state, lengths, want_state) -> (y, state or None)
PyObject* py_causal_conv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "causal_conv: seven arguments");
  const Tensor x = values("x", a[0], true), w = values("weight", a[1], true), bias = maybe("bias", a[2], true), state = maybe("state", a[4], true), lengths = maybe("lengths", a[5], true);
  const bool silu = a[3] == Py_True, want = a[6] == Py_True;
  std::pair<Tensor, Tensor> found;
  {
    const pybind11::gil_scoped_release free;
    found = causal_conv(x, w, bias, silu, state, lengths, want);
  }
  return pair_of(std::move(found));
  END_HANDLE_TH_ERRORS
}

// (x, state, weight, bias, silu, out_state) -> y
PyObject* py_causal_conv_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "causal_conv_step: six arguments");
  const Tensor x = values("x", a[0], false), state = values("state", a[1], false), w = values("weight", a[2], false), bias = maybe("bias", a[3], false), next = maybe("out_state", a[5], false);
  const bool silu = a[4] == Py_True;
  Tensor y;
  {
    const pybind11::gil_scoped_release free;
    y = causal_conv_step(x, state, w, bias, silu, next.defined() ? optional<Tensor>(next) : std::nullopt);
  }
  return object_of(std::move(y));
  END_HANDLE_TH_ERRORS
}

const char* const kScanNames[] = {"x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state", "lengths"};
bool optional_input(int i) { return i == D_ || i == Z || i == DT_BIAS || i == STATE || i == LENGTHS; }

// (x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state) -> (y, state or None)
PyObject* py_selective_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "selective_scan: twelve arguments");
  std::vector<Tensor> in;
  for (int i = 0; i <= LENGTHS; ++i) in.push_back(optional_input(i) ? maybe(kScanNames[i], a[i], true) : values(kScanNames[i], a[i], true));
  const bool softplus = a[10] == Py_True, want = a[11] == Py_True;
  std::pair<Tensor, Tensor> found;
  {
    const pybind11::gil_scoped_release free;
    found = selective_scan(std::move(in), softplus, want);
  }
  return pair_of(std::move(found));
  END_HANDLE_TH_ERRORS
}

// (x, dt, A, B, C, D, z, dt_bias, state, softplus, out_state) -> y
PyObject* py_selective_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "selective_scan_step: eleven arguments");
  std::vector<Tensor> in;
  for (int i = 0; i < INPUTS; ++i) in.push_back(optional_input(i) && i != STATE ? maybe(kScanNames[i], a[i], false) : values(kScanNames[i], a[i], false));
  const bool softplus = a[9] == Py_True;
  const Tensor next = maybe("out_state", a[10], false);
  Tensor y;
  {
    const pybind11::gil_scoped_release free;
    y = selective_scan_step(std::move(in), softplus, next.defined() ? optional<Tensor>(next) : std::nullopt);
  }
  return object_of(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (x, groups, weight, bias, eps, act) -> y
PyObject* py_group_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "group_norm: six arguments");
  const Tensor x = values("x", a[0], true), w = maybe("weight", a[2], true), b = maybe("bias", a[3], true);
  const int64_t groups = integer(a[1]), act = integer(a[5]);
  const double eps = PyFloat_AsDouble(a[4]);
  if (eps == -1 && PyErr_Occurred()) throw python_error();
  Tensor y;
  {
    const pybind11::gil_scoped_release free;
    y = group_norm(x, groups, w, b, eps, static_cast<int>(act));
  }
  return object_of(std::move(y));
  END_HANDLE_TH_ERRORS
}

#define M2_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef fast[] = {M2_FAST(causal_conv), M2_FAST(causal_conv_step), M2_FAST(selective_scan), M2_FAST(selective_scan_step), M2_FAST(group_norm), {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(_causal_calls, m) {
  m.def("bind", torch::wrap_pybind_function(bind));
  if (PyModule_AddFunctions(m.ptr(), fast) != 0) throw pybind11::error_already_set();
}
