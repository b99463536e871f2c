// CPython extension m2_amd._answer_calls: the host side of Int4Linear and token_logprobs (m2_amd/int4.py, m2_amd/scores.py).
//
// Their calls are a few microseconds of GPU time for a row or a handful of them, and checks, output tensors and the call through ctypes took
// 10 to 17 us in Python (torch's own linear: 19), a gradient 100: here the same checks raise the same errors.  us a call, one stream, back to back, Python / here:
// Int4Linear 768 x 768 11.8 / 6.3 (the launch itself 3.0, the output tensor 0.7); token_logprobs 1 x 30522 17.0 / 8.5, 128 x 30522 fp32 with its gradient 118 / 35 .. 58
// (most of it torch's own backward pass, which takes one or the other from process to process, on one machine).
#include "torch_calls.h"

namespace {

// The entry points of libm2_amd.so, which m2_amd/_lib.py has loaded.
decltype(&m2_int4_weight_bytes) int4_weight_bytes;
decltype(&m2_int4_workspace_bytes) int4_workspace_bytes;
decltype(&m2_int4_linear_fwd) int4_linear_fwd;
decltype(&m2_token_scores_workspace_bytes) token_scores_workspace_bytes;
decltype(&m2_token_scores_fwd) token_scores_fwd;
decltype(&m2_token_scores_bwd) token_scores_bwd;

void bind(const std::vector<uintptr_t>& a) {
  TORCH_CHECK(a.size() == 7, "seven addresses");
  set(last_error, a[0]);
  set(int4_weight_bytes, a[1]);
  set(int4_workspace_bytes, a[2]);
  set(int4_linear_fwd, a[3]);
  set(token_scores_workspace_bytes, a[4]);
  set(token_scores_fwd, a[5]);
  set(token_scores_bwd, a[6]);
}

// t (..., n): row r of its leading dimensions lies (r / inner) * outer + (r % inner) * row values behind the first, in t or a copy of it: one is made where
// a row's values lie apart, or the rows at more than `distances` (1 or 2) distances.
struct Rows {
  Tensor t;
  int64_t inner = 1, outer = 0, row = 0;
};
Rows rows_of(Tensor t, int distances) {
  const int64_t d = t.dim() - 1;
  if (t.is_neg()) t = t.resolve_neg();      // a view whose memory holds the negatives (the imaginary part of a conjugate)
  if (t.size(d) > 1 && t.stride(d) != 1) t = t.contiguous();
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};      // the innermost first
  int n = 0;
  for (int64_t i = d - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (n > 0 && t.stride(i) == size[n - 1] * stride[n - 1]) {
      size[n - 1] *= t.size(i);
    } else {
      if (n == distances) return rows_of(t.contiguous(), distances);
      size[n] = t.size(i), stride[n] = t.stride(i);
      ++n;
    }
  }
  return {std::move(t), size[0], n > 1 ? stride[1] : 0, stride[0]};
}

Tensor int4_linear(const Tensor& x, const Tensor& weight, int64_t N, int64_t group, const optional<Tensor>& bias, bool gelu) {
  const int type = type_of("x", x);
  TORCH_CHECK_VALUE(x.dim() > 0, "x: expected (..., K), got a single value");
  const int64_t K = x.size(-1);
  TORCH_CHECK_VALUE(N > 0 && N <= 1 << 30 && K > 0 && K <= 1 << 30, "x ", x.sizes(), " and N = ", N, ": sizes must be positive and at most 2^30");
  const auto bytes = static_cast<int64_t>(int4_weight_bytes(static_cast<int>(N), static_cast<int>(K), static_cast<int>(group)));
  TORCH_CHECK(weight.device() == x.device() && (!bias || bias->device() == x.device()), "weight and bias must live on x's device, ", x.device());
  TORCH_CHECK_VALUE(bytes > 0 && weight.scalar_type() == at::kByte && weight.is_contiguous() && weight.numel() == bytes, "weight: expected ", bytes, " bytes for (", N, ", ", K,
                    ") in groups of ", group, ", got ", weight.scalar_type(), " ", weight.sizes());
  TORCH_CHECK_VALUE(!bias || (bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->dim() == 1 && bias->numel() == N), "bias: expected float32 (", N, ")");
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  const c10::DeviceGuard guard(x.device());
  Tensor out = at::empty(shape, x.options().requires_grad(false));
  const int64_t M = x.numel() / K;
  if (M == 0) return out;
  TORCH_CHECK_VALUE(M < INT_MAX, "x: below 2^31 rows, got ", M);
  const Rows r = rows_of(x, 1);
  const auto scratch = static_cast<int64_t>(int4_workspace_bytes(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), type));
  const Tensor workspace = scratch ? at::empty({scratch}, weight.options()) : Tensor();
  const Tensor offsets = bias ? dense(*bias) : Tensor();
  check(int4_linear_fwd(r.t.data_ptr(), r.row, weight.data_ptr(), static_cast<const float*>(pointer(offsets)), out.data_ptr(), pointer(workspace), static_cast<int>(M), static_cast<int>(N),
                        static_cast<int>(K), static_cast<int>(group), gelu, type, current_stream()));
  return out;
}

// Which tokens a row may use, as the kernels read it: V bytes for all rows (row 0), or rows `row` bytes apart.
struct Allowed {
  Tensor t;
  int64_t row = 0;
};
Allowed allowed_of(const Tensor& t, int64_t V) {
  if (t.dim() == 1) return {t.contiguous(), 0};      // one list (or the only row's)
  Rows r = rows_of(t, 1);
  // rows that overlap (one list expanded to all) are one list where there is nothing else
  if (r.row == 0 && r.inner > 1) return {std::move(r.t), 0};
  if (r.inner == 1 || r.row >= V) return {std::move(r.t), std::max(V, r.row)};
  return {t.contiguous(), V};
}

// What both directions take of the arguments.
struct Scores {
  int type;
  int64_t V, rows, top_k, ignore_index;
  Tensor tokens;
  Allowed allowed;
};
Scores arguments(const Tensor& logits, const optional<Tensor>& tokens, int64_t top_k, const optional<Tensor>& allowed, int64_t ignore_index) {
  Scores s;
  s.type = type_of("logits", logits);
  TORCH_CHECK_VALUE(logits.dim() > 0 && logits.size(-1) > 0, "logits: expected (..., V), got ", logits.sizes());
  s.V = logits.size(-1);
  s.rows = logits.numel() / s.V;
  s.top_k = top_k;
  s.ignore_index = ignore_index;
  TORCH_CHECK_VALUE(s.V <= 1 << 30 && s.rows < INT_MAX, "logits: at most 2^30 values in a row and below 2^31 rows, got ", logits.sizes());
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= std::min<int64_t>(32, s.V), "top_k must lie in 0 .. ", std::min<int64_t>(32, s.V), ", got ", top_k);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  if (tokens) {
    TORCH_CHECK_VALUE(tokens->scalar_type() == at::kLong && tokens->sizes() == lead && tokens->device() == logits.device(), "tokens: expected int64 ", lead, " on ",
                      logits.device(), ", got ", tokens->scalar_type(), " ", tokens->sizes(), " on ", tokens->device());
    s.tokens = dense(*tokens);
  }
  if (allowed) {
    const bool one = allowed->dim() == 1 && allowed->size(0) == s.V;
    TORCH_CHECK_VALUE(allowed->scalar_type() == at::kBool && (one || allowed->sizes() == logits.sizes()) && allowed->device() == logits.device(), "allowed: expected bool (",
                      s.V, ") or ", logits.sizes(), " on ", logits.device(), ", got ", allowed->scalar_type(), " ", allowed->sizes(), " on ", allowed->device());
    s.allowed = allowed_of(*allowed, s.V);
  }
  return s;
}

struct Found {
  Tensor logprobs, entropy, stats, ids, top;
};
Found scores(const Tensor& logits, const Scores& s) {
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  const c10::DeviceGuard guard(logits.device());
  Found f;
  if (s.tokens.defined()) f.logprobs = at::empty(lead, f32);
  f.entropy = at::empty(lead, f32);
  f.stats = at::empty({s.rows, 2}, f32);
  if (s.top_k) {
    c10::SmallVector<int64_t, 6> shape(lead.begin(), lead.end());
    shape.push_back(s.top_k);
    f.ids = at::empty(shape, f32.dtype(at::kLong));
    f.top = at::empty(shape, f32);
  }
  if (s.rows == 0) return f;
  const Rows r = rows_of(logits, 2);
  const auto bytes = static_cast<int64_t>(token_scores_workspace_bytes(s.rows, static_cast<int>(s.V), s.type));
  const Tensor workspace = bytes ? at::empty({bytes}, f32.dtype(at::kByte)) : Tensor();
  check(token_scores_fwd(r.t.data_ptr(), static_cast<int>(r.inner), r.outer, r.row, static_cast<const long long*>(pointer(s.tokens)), s.ignore_index,
                         static_cast<const unsigned char*>(pointer(s.allowed.t)), s.allowed.row, static_cast<float*>(pointer(f.logprobs)), f.entropy.data_ptr<float>(),
                         f.stats.data_ptr<float>(), static_cast<long long*>(pointer(f.ids)), static_cast<float*>(pointer(f.top)), pointer(workspace), s.rows,
                         static_cast<int>(s.V), static_cast<int>(s.top_k), s.type, current_stream()));
  return f;
}

// A gradient of one value a row: it may be one value for all of them.
Tensor per_row(const Tensor& g) { return g.defined() ? (g.is_neg() ? g.resolve_neg() : g).reshape({-1}) : g; }

// The graph's node.  Its inputs are the gradients of entropy, log probabilities and alternatives' log probabilities, undefined where there is none.
struct TokenLogprobsBackward : torch::autograd::Node {
  SavedVariable logits_, tokens_, allowed_, entropy_, stats_, ids_;
  int type = 0;
  int64_t V = 0, rows = 0, top_k = 0, ignore_index = 0;
  bool released = false;

  std::string name() const override { return "TokenLogprobsBackward"; }

  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&logits_, &tokens_, &allowed_, &entropy_, &stats_, &ids_}) v->reset_data();
    released = true;
  }

  variable_list apply(variable_list&& g) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    // Hooks on saved tensors (torch.autograd.graph.saved_tensors_hooks) may hand out others than were saved, of another layout or anything at all.
    const Tensor logits = logits_.unpack();
    TORCH_CHECK(logits.defined() && logits.is_cuda() && logits.layout() == at::kStrided && logits.scalar_type() == (type == M2_DTYPE_F32 ? at::kFloat : at::kBFloat16) &&
                    logits.dim() > 0 && logits.size(-1) == V && logits.numel() == rows * V, "token_logprobs: the saved logits came back as other ones");
    const auto saved = [&](const char* name, Tensor t, at::ScalarType dtype, int64_t numel) {
      TORCH_CHECK(!t.defined() || (t.device() == logits.device() && t.layout() == at::kStrided && t.scalar_type() == dtype && (numel < 0 || t.numel() == numel)), "token_logprobs: the saved ",
                  name, " came back as another tensor");
      return t;
    };
    const Tensor tokens = saved("tokens", tokens_.unpack(), at::kLong, rows), allowed = saved("allowed tokens", allowed_.unpack(), at::kBool, -1),
                 entropy = saved("entropies", entropy_.unpack(shared_from_this()), at::kFloat, rows), stats = saved("sums", stats_.unpack(), at::kFloat, 2 * rows),
                 ids = saved("ids", ids_.unpack(), at::kLong, rows * top_k);
    TORCH_CHECK(!allowed.defined() || (allowed.dim() > 0 && allowed.size(-1) == V && (allowed.dim() == 1 || allowed.numel() == rows * V)),
                "token_logprobs: the saved allowed tokens came back as another tensor");
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return variable_list(1);
    Tensor grad;
    {
      const at::AutoDispatchBelowADInplaceOrView below;
      const c10::DeviceGuard guard(logits.device());
      grad = at::empty(logits.sizes(), logits.options().requires_grad(false));
      if (rows) {
        const Tensor g_h = per_row(g[0]), g_lp = per_row(g[1]), g_top = dense(g[2]);
        const Tensor token = dense(tokens), h = dense(entropy), sums = dense(stats), id = dense(ids);
        const Allowed mask = allowed.defined() ? allowed_of(allowed, V) : Allowed();
        const Rows r = rows_of(logits, 2);
        check(token_scores_bwd(r.t.data_ptr(), static_cast<int>(r.inner), r.outer, r.row, static_cast<const long long*>(pointer(token)), ignore_index,
                               static_cast<const unsigned char*>(pointer(mask.t)), mask.row, h.data_ptr<float>(), sums.data_ptr<float>(),
                               static_cast<const long long*>(pointer(id)), static_cast<const float*>(pointer(g_lp)), g_lp.defined() ? g_lp.stride(0) : 0,
                               static_cast<const float*>(pointer(g_h)), g_h.defined() ? g_h.stride(0) : 0, static_cast<const float*>(pointer(g_top)), grad.data_ptr(), V, rows,
                               static_cast<int>(V), static_cast<int>(top_k), type, current_stream()));
      }
    }
    if (at::GradMode::is_enabled()) {      // a graph of the backward pass is made: what is asked of it later has to fail
      auto node = std::make_shared<torch::autograd::DelayedError>("token_logprobs has no second derivative", 1);
      grad.set_requires_grad(true);
      grad = (*node)({grad})[0];
    }
    return {grad};
  }
};

Found scores_with_graph(const Tensor& logits, const Scores& s) {
  const std::shared_ptr<TokenLogprobsBackward> node(new TokenLogprobsBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(logits));
  Found f;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    f = scores(logits, s);
  }
  torch::autograd::set_history(variable_list{f.entropy, f.logprobs, f.top}, node);
  node->logits_ = SavedVariable(logits, false);
  node->tokens_ = SavedVariable(s.tokens, false);
  node->allowed_ = SavedVariable(s.allowed.t, false);
  node->entropy_ = SavedVariable(f.entropy, true);
  node->stats_ = SavedVariable(f.stats, false);
  node->ids_ = SavedVariable(f.ids, false);
  node->type = s.type, node->V = s.V, node->rows = s.rows, node->top_k = s.top_k, node->ignore_index = s.ignore_index;
  return f;
}

// The four results: log probabilities, entropy, ids and log probabilities of the alternatives; undefined where not asked for.
std::array<Tensor, 4> token_logprobs(const Tensor& logits, const optional<Tensor>& tokens, int64_t top_k, const optional<Tensor>& allowed, int64_t ignore_index) {
  const Scores s = arguments(logits, tokens, top_k, allowed, ignore_index);
  Found f = logits.requires_grad() && at::GradMode::is_enabled() ? scores_with_graph(logits, s) : scores(logits, s);
  return {std::move(f.logprobs), std::move(f.entropy), std::move(f.ids), std::move(f.top)};
}

// (x, weight, N, group, bias or None, gelu) -> y
PyObject* py_int4_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "int4_linear: six arguments");
  const Tensor &x = values("x", args[0], false), &weight = tensor("weight", args[1]);
  const int64_t N = integer(args[2]), group = integer(args[3]);
  const optional<Tensor> bias = args[4] == Py_None ? std::nullopt : optional<Tensor>(values("bias", args[4], false));
  const bool gelu = args[5] == Py_True;
  Tensor y;
  {
    const pybind11::gil_scoped_release free;
    y = int4_linear(x, weight, N, group, bias, gelu);
  }
  return object_of(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (logits, tokens or None, top_k, allowed or None, ignore_index) -> four results, None where not asked for
PyObject* py_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "token_logprobs: five arguments");
  const Tensor& logits = values("logits", args[0], true);
  const optional<Tensor> tokens = tensor_or_none("tokens", args[1]), allowed = tensor_or_none("allowed", args[3]);
  const int64_t top_k = integer(args[2]), ignore_index = integer(args[4]);
  std::array<Tensor, 4> found;
  {
    const pybind11::gil_scoped_release free;
    found = token_logprobs(logits, tokens, top_k, allowed, ignore_index);
  }
  auto results = pybind11::reinterpret_steal<pybind11::object>(PyTuple_New(4));
  if (!results) throw python_error();
  for (int i = 0; i < 4; ++i) {
    PyObject* o = object_of(std::move(found[i]));
    if (!o) throw python_error();
    PyTuple_SET_ITEM(results.ptr(), i, o);
  }
  return results.release().ptr();
  END_HANDLE_TH_ERRORS
}

PyMethodDef fast[] = {
    {"int4_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_int4_linear)), METH_FASTCALL, nullptr},
    {"token_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_token_logprobs)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PYBIND11_MODULE(_answer_calls, m) {
  m.def("bind", torch::wrap_pybind_function(bind));
  if (PyModule_AddFunctions(m.ptr(), fast) != 0) throw pybind11::error_already_set();
}
