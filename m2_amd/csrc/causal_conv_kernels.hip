// The short causal convolution of a mixer on hidden states whose channels lie last, its gradient, and the same for one token.
//
//   pre[t, c] = bias[c] + sum_k w[c, k] x[t - K + 1 + k, c]      y = pre, or pre sigmoid(pre)      x[t] for t < 0: the state, oldest first, or 0
//   g = gy act'(pre)     gx[s] = sum_j w[K - 1 - j] g[s + j]     gw[k] = sum g[t] x[t - K + 1 + k]     gb = sum g
//
// A thread owns V neighbouring channels and a run of positions; what the taps need of the positions before stays in registers, so that x is read once but for the ends of runs.  Bound by memory: 4 x
// 8192 x 1536 bf16 47 us (4.3 TB/s, where a copy of as much reaches 5.1), 8 x 2049 x 1920 fp32 with its gradient 118 (4.3 TB/s; the forward 37, the gradient 66, its sums over runs 5).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "lane_ops.h"

namespace m2 {

constexpr int kMaxTaps = 8;

struct ConvArgs {
  const void* x;
  long x_batch, x_row;
  const float *w, *bias;             // (C, K), (C) or null
  const void* state;                 // (B, K - 1, C) or null
  const long long* lengths;          // (B) or null
  void *y, *state_out;               // (B, L, C), (B, K - 1, C) or null
  int B, L, C, K, silu;
  int run, runs, columns;            // positions a thread, runs of a sequence, vectors of channels
  // gradients
  const void* gy;
  long gy_batch, gy_row;
  const void* gstate_out;            // or null
  void *gx, *gstate;                 // or null
  float* partials;                   // (workgroups along runs, K + 1, C) or null
};

__device__ __forceinline__ int length_of(const long long* lengths, int b, int L) {
  if (!lengths) return L;
  const long long n = lengths[b];
  return n < 0 ? 0 : n > L ? L : (int)n;
}

// The weights of V channels, the last tap last.
template <int V, int K>
__device__ __forceinline__ void load_taps(const float* w, const float* bias, long c, float (&taps)[K][V], float (&b)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) taps[k][v] = w[(c + v) * K + k];
    b[v] = bias ? bias[c + v] : 0.f;
  }
}

// Position t of a sequence of n, of its state for t < 0 (as far as it goes back), 0 elsewhere.
template <typename T, int V, int K>
__device__ __forceinline__ void load_position(const ConvArgs& p, int b, int t, long c, int n, float (&f)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = 0.f;
  if (t >= 0 && t < n) {
    load_values<T, V>(static_cast<const T*>(p.x) + b * p.x_batch + t * p.x_row + c, f);
  } else if (t < 0 && t >= 1 - K && p.state) {
    load_values<T, V>(static_cast<const T*>(p.state) + ((long)b * (K - 1) + t + K - 1) * p.C + c, f);
  }
}
// Positions t .. t + U - 1 below `end`, asked for together where all of them are inside the sequence.
template <typename T, int V, int K, int U>
__device__ __forceinline__ void load_positions(const ConvArgs& p, int b, int t, int end, long c, int n, float (*f)[V]) {
  if (t >= 0 && t + U <= end && t + U <= n) {
    const T* x = static_cast<const T*>(p.x) + b * p.x_batch + t * p.x_row + c;
#pragma unroll
    for (int u = 0; u < U; ++u) load_values<T, V>(x + u * p.x_row, f[u]);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) load_position<T, V, K>(p, b, t + u < end ? t + u : n, c, n, f[u]);
  }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvArgs p) {
  constexpr int U = 8;      // positions asked for together
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t run = i / (uint32_t)p.columns;
  if (run >= (uint32_t)p.runs) return;
  const int b = blockIdx.y;
  const long c = (long)(i - run * (uint32_t)p.columns) * V;
  const int n = length_of(p.lengths, b, p.L), t0 = run * p.run, t1 = min(t0 + p.run, p.L);
  float taps[K][V], bias[V];
  load_taps<V, K>(p.w, p.bias, c, taps, bias);
  float win[K - 1 + U][V];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) load_position<T, V, K>(p, b, t0 - (K - 1) + k, c, n, win[k]);
  T* y = static_cast<T*>(p.y) + ((long)b * p.L) * p.C + c;
  for (int t = t0; t < t1; t += U) {
    load_positions<T, V, K, U>(p, b, t, t1, c, n, win + K - 1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float out[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s = bias[v];
#pragma unroll
        for (int k = 0; k < K; ++k) s = fmaf(taps[k][v], win[u + k][v], s);
        s = p.silu ? silu<T>(s) : s;
        out[v] = t + u < n ? s : 0.f;
      }
      if (t + u < t1) store_values<T, V>(y + (long)(t + u) * p.C, out);
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) win[k][v] = win[U + k][v];
  }
  if (run == 0 && p.state_out) {
    for (int k = 0; k < K - 1; ++k) {
      float f[V];
      load_position<T, V, K>(p, b, n - (K - 1) + k, c, n, f);
      store_values<T, V>(static_cast<T*>(p.state_out) + ((long)b * (K - 1) + k) * p.C + c, f);
    }
  }
}

// Lanes of a workgroup: `CL` vectors of channels times 256 / CL runs, whose sums for the weights' gradients are joined in shared memory.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void causal_conv_bwd_kernel(ConvArgs p, int CL) {
  constexpr int U = 4;
  extern __shared__ float shared[];      // (256 / CL, K + 1, CL, V)
  const int lane = threadIdx.x % CL, part = threadIdx.x / CL, parts = 256 / CL;
  const int column = blockIdx.y * CL + lane;
  const long job = (long)blockIdx.x * parts + part;      // (sequence, run)
  const bool on = column < p.columns && job < (long)p.B * p.runs;
  const int b = on ? job / p.runs : 0, run = on ? job - (long)b * p.runs : 0;
  const long c = on ? (long)column * V : 0;
  float gw[K][V], gb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    gb[v] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) gw[k][v] = 0.f;
  }
  if (on) {
    const int n = length_of(p.lengths, b, p.L), t0 = run * p.run, t1 = min(t0 + p.run, p.L);
    const int s0 = run == 0 && p.gstate ? t0 - (K - 1) : t0;      // first position whose gradient is written
    float taps[K][V], bias[V], x[K - 1 + U][V], g[K - 1 + U][V];      // position t + u at K - 1 + u
    load_taps<V, K>(p.w, p.bias, c, taps, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      load_position<T, V, K>(p, b, s0 - (K - 1) + k, c, n, x[k]);
#pragma unroll
      for (int v = 0; v < V; ++v) g[k][v] = 0.f;
    }
    const T* gy = static_cast<const T*>(p.gy) + b * p.gy_batch + c;
    const int end = t1 + K - 1;
    for (int t = s0; t < end; t += U) {
      load_positions<T, V, K, U>(p, b, t, end, c, n, x + K - 1);
      if (t >= 0 && t + U <= end && t + U <= n) {
#pragma unroll
        for (int u = 0; u < U; ++u) load_values<T, V>(gy + (t + u) * p.gy_row, g[K - 1 + u]);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int v = 0; v < V; ++v) g[K - 1 + u][v] = 0.f;
          if (t + u >= 0 && t + u < n && t + u < end) load_values<T, V>(gy + (t + u) * p.gy_row, g[K - 1 + u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = t + u;
        const bool inside = at >= 0 && at < n;
        if (p.silu) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float pre = bias[v];
#pragma unroll
            for (int k = 0; k < K; ++k) pre = fmaf(taps[k][v], x[u + k][v], pre);
            const float slope = silu_slope<T>(pre);
            g[K - 1 + u][v] = inside ? g[K - 1 + u][v] * slope : 0.f;
          }
        }
        if (at >= t0 && at < t1 && inside) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            gb[v] += g[K - 1 + u][v];
#pragma unroll
            for (int k = 0; k < K; ++k) gw[k][v] = fmaf(g[K - 1 + u][v], x[u + k][v], gw[k][v]);
          }
        }
        const int s = at - (K - 1);      // g[u ..] = positions s .. at
        if (s < s0 || s >= t1) continue;
        float out[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < K; ++j) sum = fmaf(taps[K - 1 - j][v], g[u + j][v], sum);
          out[v] = s < n ? sum : 0.f;
        }
        const int kept = s - (n - (K - 1));      // its place in the state that the sequence ends with
        if (p.gstate_out && kept >= 0 && kept < K - 1) {
          float more[V];
          load_values<T, V>(static_cast<const T*>(p.gstate_out) + ((long)b * (K - 1) + kept) * p.C + c, more);
#pragma unroll
          for (int v = 0; v < V; ++v) out[v] += more[v];
        }
        if (s >= 0) {
          if (p.gx) store_values<T, V>(static_cast<T*>(p.gx) + ((long)b * p.L + s) * p.C + c, out);
        } else {
          store_values<T, V>(static_cast<T*>(p.gstate) + ((long)b * (K - 1) + s + K - 1) * p.C + c, out);
        }
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) x[k][v] = x[U + k][v], g[k][v] = g[U + k][v];
    }
  }
  if (!p.partials) return;
  float* mine = shared + ((long)part * (K + 1) * CL + lane) * V;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) mine[k * CL * V + v] = gw[k][v];
    mine[K * CL * V + v] = gb[v];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < (K + 1) * CL * V; j += 256) {
    const int k = j / (CL * V), at = j % (CL * V);
    const long channel = (long)blockIdx.y * CL * V + at;
    if (channel >= p.C) continue;
    float sum = 0.f;
    for (int q = 0; q < parts; ++q) sum += shared[(q * (K + 1) + k) * CL * V + at];
    p.partials[((long)blockIdx.x * (K + 1) + k) * p.C + channel] = sum;
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(ConvArgs p) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, b = i / (uint32_t)p.columns;
  if (b >= (uint32_t)p.B) return;
  const long c = (long)(i - b * (uint32_t)p.columns) * V;
  const int K = p.K;
  const T* old = static_cast<const T*>(p.state) + (long)b * (K - 1) * p.C + c;
  T* kept = static_cast<T*>(p.state_out) + (long)b * (K - 1) * p.C + c;
  float rows[kMaxTaps][V], s[V];
#pragma unroll
  for (int k = 0; k < kMaxTaps; ++k) {
    if (k < K - 1) load_values<T, V>(old + (long)k * p.C, rows[k]);
    else if (k == K - 1) load_values<T, V>(static_cast<const T*>(p.x) + b * p.x_batch + c, rows[k]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = p.bias ? p.bias[c + v] : 0.f;
#pragma unroll
  for (int k = 0; k < kMaxTaps; ++k) {
    if (k >= K) break;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = fmaf(p.w[(c + v) * K + k], rows[k][v], s[v]);
    if (k > 0) store_values<T, V>(kept + (long)(k - 1) * p.C, rows[k]);
  }
  if (p.silu) {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = silu<T>(s[v]);
  }
  store_values<T, V>(static_cast<T*>(p.y) + (long)b * p.C + c, s);
}

// A workgroup sums 64 columns, 16 threads a column with eight rows on their way each, over all rows of the partial results.
__global__ __launch_bounds__(1024) void sum_partials_kernel(const float* __restrict__ partials, long rows, int K, long n, float* wide, float* last) {
  constexpr int U = 8;
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, planes = last ? K + 1 : K;
  const long width = n * (K + 1), at = blockIdx.x * 64L + lane;
  float sums[U], sum = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) sums[u] = 0.f;
  if (at < n * planes) {
    for (long r = w; r < rows; r += 16 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = partials[min(r + 16 * u, rows - 1) * width + at];
#pragma unroll
      for (int u = 0; u < U; ++u) sums[u] += r + 16 * u < rows ? v[u] : 0.f;
    }
  }
  part[w][lane] = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
  __syncthreads();
  if (w == 0 && at < n * planes) {
    sum = 0.f;
#pragma unroll
    for (int o = 0; o < 16; ++o) sum += part[o][lane];
    const long k = at / n, j = at - k * n;
    if (k < K) {
      if (wide) wide[j * K + k] = sum;
    } else {
      last[j] = sum;
    }
  }
}

int sum_partials(const float* partials, long rows, int K, long n, float* wide, float* last, hipStream_t stream) {
  const long columns = n * (last ? K + 1 : K);
  if (columns == 0) return M2_OK;
  hipLaunchKernelGGL(sum_partials_kernel, dim3((unsigned)((columns + 63) / 64)), dim3(1024), 0, stream, partials, rows, K, n, wide, last);
  return check_launch("sum_partials_kernel");
}

namespace {

// Values a thread moves at a time: 16 bytes where rows and pointers allow it.
template <typename T>
int vector_of(int C, std::initializer_list<const void*> pointers, std::initializer_list<long> strides, int most) {
  uintptr_t bits = 0;
  for (const void* q : pointers) bits |= (uintptr_t)q;
  for (long s : strides) bits |= (uintptr_t)(s * (long)sizeof(T));
  bits |= (uintptr_t)((long)C * (long)sizeof(T));
  for (int v = most; v > 1; v /= 2)
    if (bits % (v * sizeof(T)) == 0) return v;
  return 1;
}

// sequences: the most that the call's grid holds
int check_sizes(const char* name, int B, int L, int C, int K, int dtype, int sequences = 65535) {
  if (B < 1 || L < 1 || C < 1 || B > sequences) return set_error(M2_ERR_ARG, "%s: B=%d (1 .. %d), L=%d, C=%d", name, B, sequences, L, C);
  if (K < 1 || K > kMaxTaps) return set_error(M2_ERR_UNSUPPORTED, "%s: K=%d taps, 1 .. %d are supported", name, K, kMaxTaps);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype %d", name, dtype);
  if (C > 1 << 20 || L > 1 << 30 || (long)B * L > (1L << 36) / C) return set_error(M2_ERR_ARG, "%s: at most 2^20 channels, 2^30 positions and 2^36 values", name);
  return M2_OK;
}

// f(number of taps as a constant)
template <typename F>
void with_taps(int K, F&& f) {
  switch (K) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}

template <typename T, int V>
int launch_fwd(const ConvArgs& p, hipStream_t stream) {
  const long threads = (long)p.columns * p.runs;
  const dim3 grid((unsigned)((threads + 255) / 256), p.B);
  with_taps(p.K, [&](auto k) { hipLaunchKernelGGL((causal_conv_kernel<T, V, decltype(k)::value>), grid, dim3(256), 0, stream, p); });
  return check_launch("causal_conv_kernel");
}

// Positions a thread takes: 32, of which the K - 1 ahead are read twice, or fewer where that leaves a compute unit below 512 threads.  4 x 8192 x 1536 bf16, us with 8 / 16 / 32 positions
// and four channels a thread: 51.4 / 47.5 / 47.3 (4.25 TB/s); eight channels: 67 / 53.5 / 49.2; 8 x 2049 x 1920 fp32 with its gradient 136 / 124 / 122 (4.1 TB/s).
int run_of(int B, int L, long columns) {
  int run = 32;
  while (run > 8 && columns * B * ((L + run - 1) / run) < 512L * num_cus()) run /= 2;
  return run;
}

template <typename T>
int fwd(ConvArgs p, hipStream_t stream) {
  int V = vector_of<T>(p.C, {p.x, p.state, p.y, p.state_out}, {p.x_batch, p.x_row}, 4);
  if (V < 4) V = 1;
  p.columns = p.C / V;
  p.run = run_of(p.B, p.L, p.columns);
  p.runs = (p.L + p.run - 1) / p.run;
  return V == 4 ? launch_fwd<T, 4>(p, stream) : launch_fwd<T, 1>(p, stream);
}

struct BwdPlan {
  int V, CL, run, runs;
  long rows;      // of partial sums
};
BwdPlan bwd_plan(int B, int L, int C, int V) {
  BwdPlan r;
  r.V = V;
  const int columns = C / V;
  r.CL = 64;
  while (r.CL > 8 && r.CL / 2 >= columns) r.CL /= 2;
  r.run = run_of(B, L, columns);
  r.runs = (L + r.run - 1) / r.run;
  r.rows = ((long)B * r.runs + 256 / r.CL - 1) / (256 / r.CL);
  return r;
}

template <typename T, int V>
int launch_bwd(const ConvArgs& p, const BwdPlan& plan, hipStream_t stream) {
  const dim3 grid((unsigned)plan.rows, (p.columns + plan.CL - 1) / plan.CL);
  const size_t lds = p.partials ? sizeof(float) * 256 * (p.K + 1) * V : 0;
  with_taps(p.K, [&](auto k) { hipLaunchKernelGGL((causal_conv_bwd_kernel<T, V, decltype(k)::value>), grid, dim3(256), lds, stream, p, plan.CL); });
  return check_launch("causal_conv_bwd_kernel");
}

template <typename T>
int bwd(ConvArgs p, float* gw, float* gb, float* workspace, hipStream_t stream) {
  const int V = vector_of<T>(p.C, {p.x, p.state, p.gy, p.gstate_out, p.gx, p.gstate}, {p.x_batch, p.x_row, p.gy_batch, p.gy_row}, 4) == 4 ? 4 : 1;
  const BwdPlan plan = bwd_plan(p.B, p.L, p.C, V);
  if (plan.rows >= 1L << 24) return set_error(M2_ERR_ARG, "causal_conv_bwd: B=%d sequences of L=%d are more than a launch holds", p.B, p.L);
  p.columns = p.C / V;
  p.run = plan.run, p.runs = plan.runs;
  p.partials = gw || gb ? workspace : nullptr;
  const int rc = V == 4 ? launch_bwd<T, 4>(p, plan, stream) : launch_bwd<T, 1>(p, plan, stream);
  if (rc != M2_OK || !p.partials) return rc;
  return sum_partials(workspace, plan.rows, p.K, p.C, gw, gb, stream);
}

}  // namespace
}  // namespace m2

using namespace m2;

extern "C" int m2_causal_conv_fwd(const void* x, long x_batch, long x_row, const float* w, const float* bias, const void* state, const long long* lengths, void* y, void* state_out,
                                  int B, int L, int C, int K, int silu, int dtype, void* stream) {
  if (!x || !w || !y) return set_error(M2_ERR_ARG, "causal_conv_fwd: null pointer");
  if (int rc = check_sizes("causal_conv_fwd", B, L, C, K, dtype)) return rc;
  ConvArgs p{};
  p.x = x, p.x_batch = x_batch, p.x_row = x_row, p.w = w, p.bias = bias, p.state = state, p.lengths = lengths, p.y = y, p.state_out = state_out;
  p.B = B, p.L = L, p.C = C, p.K = K, p.silu = silu;
  return dtype == M2_DTYPE_F32 ? fwd<float>(p, (hipStream_t)stream) : fwd<uint16_t>(p, (hipStream_t)stream);
}

extern "C" size_t m2_causal_conv_bwd_workspace_bytes(int B, int L, int C, int K, int dtype) {
  if (check_sizes("causal_conv_bwd", B, L, C, K, dtype)) return 0;
  // the most that either width needs
  const long rows = std::max(C % 4 == 0 ? bwd_plan(B, L, C, 4).rows : 0, bwd_plan(B, L, C, 1).rows);
  return sizeof(float) * (size_t)rows * (K + 1) * C;
}

extern "C" int m2_causal_conv_bwd(const void* x, long x_batch, long x_row, const float* w, const float* bias, const void* state, const long long* lengths, const void* gy,
                                  long gy_batch, long gy_row, const void* gstate_out, void* gx, float* gw, float* gb, void* gstate, void* workspace, int B, int L, int C, int K,
                                  int silu, int dtype, void* stream) {
  if (!x || !w || !gy || ((gw || gb) && !workspace)) return set_error(M2_ERR_ARG, "causal_conv_bwd: null pointer");
  if (int rc = check_sizes("causal_conv_bwd", B, L, C, K, dtype)) return rc;
  ConvArgs p{};
  p.x = x, p.x_batch = x_batch, p.x_row = x_row, p.w = w, p.bias = bias, p.state = state, p.lengths = lengths;
  p.gy = gy, p.gy_batch = gy_batch, p.gy_row = gy_row, p.gstate_out = gstate_out, p.gx = gx, p.gstate = gstate;
  p.B = B, p.L = L, p.C = C, p.K = K, p.silu = silu;
  float* ws = static_cast<float*>(workspace);
  return dtype == M2_DTYPE_F32 ? bwd<float>(p, gw, gb, ws, (hipStream_t)stream) : bwd<uint16_t>(p, gw, gb, ws, (hipStream_t)stream);
}

extern "C" int m2_causal_conv_step(const void* x, long x_batch, const void* state, const float* w, const float* bias, void* y, void* state_out, int B, int C, int K, int silu, int dtype,
                                   void* stream) {
  if (!x || !w || !y || (K > 1 && (!state || !state_out))) return set_error(M2_ERR_ARG, "causal_conv_step: null pointer");
  if (int rc = check_sizes("causal_conv_step", B, 1, C, K, dtype, 1 << 30)) return rc;
  if ((long)B * C > 1L << 31) return set_error(M2_ERR_ARG, "causal_conv_step: at most 2^31 values");
  ConvArgs p{};
  p.x = x, p.x_batch = x_batch, p.w = w, p.bias = bias, p.state = state, p.y = y, p.state_out = state_out;
  p.B = B, p.L = 1, p.C = C, p.K = K, p.silu = silu;
  const auto launch = [&](auto t) {
    using T = decltype(t);
    const bool wide = vector_of<T>(C, {x, state, y, state_out}, {x_batch}, 2) == 2;
    p.columns = wide ? C / 2 : C;
    const dim3 grid((unsigned)(((long)p.columns * B + 255) / 256));
    if (wide) hipLaunchKernelGGL((causal_conv_step_kernel<T, 2>), grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((causal_conv_step_kernel<T, 1>), grid, dim3(256), 0, (hipStream_t)stream, p);
    return check_launch("causal_conv_step_kernel");
  };
  return dtype == M2_DTYPE_F32 ? launch(float{}) : launch(uint16_t{});
}
