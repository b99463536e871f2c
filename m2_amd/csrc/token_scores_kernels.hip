// What a masked-LM head's logits say about given tokens: log probability, entropy, the most likely alternatives, and the gradient of the three.
//
//   z_j = x_j where token j is allowed, -inf elsewhere     m = max z     s = sum exp(z_j - m)     lp_j = z_j - m - log s     p_j = exp(lp_j)
//   H = -sum p_j lp_j = log s - sum exp(z_j - m) (z_j - m) / s
//   dx_j = sum over the outputs of g ([j is its token] - p_j) - g_H p_j (lp_j + H), 0 where z_j = -inf
//
// One pass over a row: every thread keeps the largest value it has met and both sums relative to it, and rescales them when a larger one comes.
// The largest value itself, and differences to it, are kept (and not products with log2 e, which overflow for a mask of the type's lowest value).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "m2_internal.h"

namespace m2 {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxTop = 32;
constexpr long kMaxGrid = 1 << 20;      // workgroups of a launch; what is left of the rows they take in turn
constexpr float kNegInf = -__builtin_inff();

// The rows of logits: row r starts (r / inner) * outer + (r % inner) * row values behind the first.
struct LogitRows {
  const void* x;
  long outer, row;
  int inner;
  const unsigned char* allowed;      // or null: all
  long allowed_row;                  // 0: one list for all rows
};

// Sixteen bytes of a row, at any address of its type: rows of an odd vocabulary start anywhere.
typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) u32x4_any;
typedef uint32_t __attribute__((ext_vector_type(2), aligned(1))) u32x2_any;
typedef uint32_t __attribute__((aligned(1))) u32_any;

template <typename T> struct Row;
template <> struct Row<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(const void* p, long i) { return reinterpret_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ void unpack(const u32x4_any& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ u32x4_any pack(const float (&f)[4]) {
    return u32x4_any{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
  }
  static __device__ __forceinline__ void put(void* p, long i, float f) { reinterpret_cast<float*>(p)[i] = f; }
  static __device__ __forceinline__ void masks(const unsigned char* a, float (&f)[4]) {
    const uint32_t b = *reinterpret_cast<const u32_any*>(a);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (b >> (8 * i)) & 0xff ? f[i] : kNegInf;
  }
};
template <> struct Row<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(const void* p, long i) { return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]); }
  static __device__ __forceinline__ void unpack(const u32x4_any& v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4_any pack(const float (&f)[8]) {
    return u32x4_any{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  }
  static __device__ __forceinline__ void put(void* p, long i, float f) { reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16(f); }
  static __device__ __forceinline__ void masks(const unsigned char* a, float (&f)[8]) {
    const u32x2_any b = *reinterpret_cast<const u32x2_any*>(a);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (b[i / 4] >> (8 * (i % 4))) & 0xff ? f[i] : kNegInf;
  }
};

template <typename T>
__device__ __forceinline__ const char* row_of(const LogitRows& in, long r) {
  return reinterpret_cast<const char*>(in.x) + ((r / in.inner) * in.outer + (r % in.inner) * in.row) * (long)sizeof(T);
}

template <typename T, bool MASK>
__device__ __forceinline__ float value_at(const char* x, const unsigned char* a, long j) {
  const float v = Row<T>::one(x, j);
  return MASK && !a[j] ? kNegInf : v;
}

// The hardware's 2^x: one ulp, results below 2^-126 are 0.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum, sum of exp(z - m) and sum of exp(z - m) (z - m).
struct Sums {
  float m = kNegInf, s = 0.f, t = 0.f;
};

// What sums relative to `from` become relative to `to` >= from.  Differences below -1e4 stand for all that exp takes to zero, -inf and
// (-inf) - (-inf) among them, so that nothing times zero is NaN; a NaN in the sums stays one.
__device__ __forceinline__ void rescale(Sums& a, float to) {
  const float d = fmaxf(a.m - to, -1e4f), f = exp2_(d * kLog2e);
  a.t = f * fmaf(d, a.s, a.t);
  a.s *= f;
  a.m = to;
}

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m);
  rescale(b, m);
  return {m, a.s + b.s, a.t + b.t};
}

template <int N>
__device__ __forceinline__ void add_values(Sums& a, const float (&z)[N]) {
  float c = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) c = fmaxf(c, z[i]);
  if (c > a.m) rescale(a, c);
  const float base = a.m == kNegInf ? 0.f : a.m;      // nothing but -inf (and NaN, which has to show) so far
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = z[i] - base, e = exp2_(d * kLog2e);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e4f), a.t);
  }
}

// (value, id) before (other, other_id): larger value first, then the lower id.
__device__ __forceinline__ bool before(float v, int id, float w, int wid) { return v > w || (v == w && id < wid); }

template <typename T, bool MASK>
__global__ __launch_bounds__(256) void token_scores_kernel(LogitRows in, const long long* __restrict__ tokens, long long ignore_index,
                                                           float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ stats,
                                                           long long* __restrict__ top_ids, float* __restrict__ top_logprobs, long rows, int V, int top_k) {
  constexpr int N = Row<T>::N;
  __shared__ float part_m[4], part_s[4], part_t[4];
  __shared__ float best_v[4];
  __shared__ int best_i[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const char* x = row_of<T>(in, r);
    const unsigned char* a = MASK ? in.allowed + r * in.allowed_row : nullptr;
    const int nvec = V / N;
    Sums mine;
    for (int i = tid; i < nvec; i += 256) {
      float z[N];
      Row<T>::unpack(*reinterpret_cast<const u32x4_any*>(x + (long)i * 16), z);
      if (MASK) Row<T>::masks(a + (long)i * N, z);
      add_values<N>(mine, z);
    }
    if (nvec * N + tid < V) {
      const float z[1] = {value_at<T, MASK>(x, a, nvec * N + tid)};
      add_values<1>(mine, z);
    }
    for (int o = 32; o > 0; o >>= 1) mine = join(mine, Sums{__shfl_xor(mine.m, o), __shfl_xor(mine.s, o), __shfl_xor(mine.t, o)});
    if (lane == 0) part_m[wave] = mine.m, part_s[wave] = mine.s, part_t[wave] = mine.t;
    __syncthreads();
    const auto part = [&](int w) { return Sums{part_m[w], part_s[w], part_t[w]}; };
    const Sums all = join(join(part(0), part(1)), join(part(2), part(3)));
    const bool empty = all.s == 0.f;
    const float logs = empty ? 0.f : logf(all.s);
    const bool broken = all.s != all.s;          // a NaN or +inf among the values
    if (tid == 0) {
      if (tokens) {
        const long long t = tokens[r];
        float lp = 0.f;
        if (t != ignore_index) {
          if (t < 0 || t >= V) lp = __builtin_nanf("");
          else {
            const float z = value_at<T, MASK>(x, a, t);
            lp = broken ? __builtin_nanf("") : z == kNegInf ? kNegInf : (z - all.m) - logs;
          }
        }
        logprobs[r] = lp;
      }
      entropy[r] = empty ? 0.f : logs - all.t / all.s;
      stats[2 * r] = broken ? __builtin_nanf("") : all.m;
      stats[2 * r + 1] = logs;
    }
    // the alternatives one after the other: the first of those behind the last one
    float last_v = __builtin_inff();
    int last_i = -1;
    for (int k = 0; k < top_k; ++k) {
      float bv = kNegInf;
      int bi = 0x7fffffff;
      if (!broken)
        for (int j = tid; j < V; j += 256) {
          const float v = value_at<T, MASK>(x, a, j);
          if (before(last_v, last_i, v, j) && before(v, j, bv, bi)) bv = v, bi = j;
        }
      for (int o = 32; o > 0; o >>= 1) {
        const float ov = __shfl_xor(bv, o);
        const int oi = __shfl_xor(bi, o);
        if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
      }
      if (lane == 0) best_v[wave] = bv, best_i[wave] = bi;
      __syncthreads();
      for (int w = 0; w < 4; ++w)
        if (before(best_v[w], best_i[w], bv, bi)) bv = best_v[w], bi = best_i[w];
      __syncthreads();
      if (tid == 0) {
        const bool none = broken || bv == kNegInf;
        top_ids[r * top_k + k] = none ? -1 : bi;
        top_logprobs[r * top_k + k] = broken ? __builtin_nanf("") : none ? kNegInf : (bv - all.m) - logs;
      }
      last_v = bv;
      last_i = bi;
    }
    __syncthreads();      // the row's shared values have been read
  }
}

struct ScoreGrads {
  const float *logprobs, *entropy, *top;      // any of them null: not asked for
  long logprobs_stride, entropy_stride;       // 0: one value for all rows
};

constexpr int kBwdChunk = 4;      // vectors of a thread

template <typename T, bool MASK>
__global__ __launch_bounds__(256) void token_scores_grad_kernel(LogitRows in, const long long* __restrict__ tokens, long long ignore_index,
                                                                const float* __restrict__ entropy, const float* __restrict__ stats,
                                                                const long long* __restrict__ top_ids, ScoreGrads g, char* __restrict__ grad,
                                                                long grad_row, long rows, int V, int top_k) {
  constexpr int N = Row<T>::N;
  __shared__ int ids[kMaxTop + 1];
  __shared__ float gs[kMaxTop + 1];
  const int tid = threadIdx.x;
  for (long r = blockIdx.y; r < rows; r += gridDim.y) {
    const char* x = row_of<T>(in, r);
    const unsigned char* a = MASK ? in.allowed + r * in.allowed_row : nullptr;
    char* out = grad + r * grad_row * (long)sizeof(T);
    const float m = stats[2 * r], logs = stats[2 * r + 1];
    const bool empty = m == kNegInf;
    // the outputs' tokens and gradients
    if (tid <= top_k) {
      int id = -1;
      float v = 0.f;
      if (tid < top_k) {
        if (g.top) id = (int)top_ids[r * top_k + tid], v = id < 0 ? 0.f : g.top[r * top_k + tid];
      } else if (tokens && g.logprobs) {
        const long long t = tokens[r];
        if (t != ignore_index) {
          const bool bad = t < 0 || t >= V;
          id = bad ? -1 : (int)t;
          v = bad ? __builtin_nanf("") : g.logprobs[r * g.logprobs_stride];
        }
      }
      ids[tid] = id;
      gs[tid] = v;
    }
    __syncthreads();
    float total = 0.f;
    for (int e = 0; e <= top_k; ++e) total += gs[e];
    const float gh = g.entropy ? g.entropy[r * g.entropy_stride] : 0.f, h = entropy[r];
    const auto slope = [&](float z) {
      if (z == kNegInf || empty) return 0.f;
      const float lp = (z - m) - logs;
      return -exp2_(lp * kLog2e) * fmaf(gh, fmaxf(lp, -1e4f) + h, total);
    };
    const int nvec = V / N, first = (int)blockIdx.x * 256 * kBwdChunk, lo = first * N;
  #pragma unroll
    for (int c = 0; c < kBwdChunk; ++c) {
      const int i = first + c * 256 + tid;
      if (i < nvec) {
        float z[N];
        Row<T>::unpack(*reinterpret_cast<const u32x4_any*>(x + (long)i * 16), z);
        if (MASK) Row<T>::masks(a + (long)i * N, z);
  #pragma unroll
        for (int n = 0; n < N; ++n) z[n] = slope(z[n]);
        *reinterpret_cast<u32x4_any*>(out + (long)i * 16) = Row<T>::pack(z);
      }
    }
    const bool last = blockIdx.x == gridDim.x - 1;
    if (last && nvec * N + tid < V) Row<T>::put(out, nvec * N + tid, slope(value_at<T, MASK>(x, a, nvec * N + tid)));
    __syncthreads();
    // the tokens themselves: what the whole row's pass wrote there lacks the outputs' own gradients
    const int hi = last ? V : lo + 256 * kBwdChunk * N;
    if (tid <= top_k && ids[tid] >= lo && ids[tid] < hi) {
      const int id = ids[tid];
      float own = 0.f;
      for (int e = 0; e <= top_k; ++e) own += ids[e] == id ? gs[e] : 0.f;
      const float z = value_at<T, MASK>(x, a, id);
      Row<T>::put(out, id, z == kNegInf || empty ? 0.f : slope(z) + own);
    }
    __syncthreads();      // ids and gs have been read
  }
}

static int check_rows(const char* who, const void* logits, int inner, long outer, long row, const unsigned char* allowed, long allowed_row, long rows,
                      int V, int top_k, int dtype) {
  if (!logits) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype must be M2_DTYPE_F32 or M2_DTYPE_BF16 (got %d)", who, dtype);
  if (rows <= 0 || V <= 0 || inner <= 0 || outer < 0 || row < 0) return set_error(M2_ERR_ARG, "%s: rows=%ld V=%d inner=%d outer=%ld row=%ld", who, rows, V, inner, outer, row);
  if (V > (1 << 30)) return set_error(M2_ERR_UNSUPPORTED, "%s: at most 2^30 values in a row (V=%d)", who, V);
  if (top_k < 0 || top_k > kMaxTop || top_k > V) return set_error(M2_ERR_UNSUPPORTED, "%s: 0 to %d alternatives, at most V (top_k=%d V=%d)", who, kMaxTop, top_k, V);
  if (allowed && allowed_row != 0 && allowed_row < V) return set_error(M2_ERR_ARG, "%s: allowed_row=%ld is less than V=%d", who, allowed_row, V);
  if ((uintptr_t)logits % (dtype == M2_DTYPE_F32 ? 4 : 2)) return set_error(M2_ERR_UNSUPPORTED, "%s: logits must be aligned to their type", who);
  return M2_OK;
}

}  // namespace m2

using namespace m2;

extern "C" int m2_token_scores_fwd(const void* logits, int inner, long outer_stride, long row_stride, const long long* tokens, long long ignore_index,
                                   const unsigned char* allowed, long allowed_row, float* logprobs, float* entropy, float* stats, long long* top_ids,
                                   float* top_logprobs, long rows, int V, int top_k, int dtype, void* stream) {
  const char* who = "m2_token_scores_fwd";
  if (int rc = check_rows(who, logits, inner, outer_stride, row_stride, allowed, allowed_row, rows, V, top_k, dtype)) return rc;
  if (!entropy || !stats || (tokens && !logprobs) || (top_k && (!top_ids || !top_logprobs))) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  const LogitRows in = {logits, outer_stride, row_stride, inner, allowed, allowed_row};
  hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows < kMaxGrid ? rows : kMaxGrid)), dim3(256), 0, st, in, tokens, ignore_index, logprobs, entropy, stats, top_ids, top_logprobs,
                       rows, V, top_k);
  };
  if (dtype == M2_DTYPE_F32) allowed ? go(token_scores_kernel<float, true>) : go(token_scores_kernel<float, false>);
  else allowed ? go(token_scores_kernel<uint16_t, true>) : go(token_scores_kernel<uint16_t, false>);
  return check_launch("token_scores");
}

extern "C" int m2_token_scores_bwd(const void* logits, int inner, long outer_stride, long row_stride, const long long* tokens, long long ignore_index,
                                   const unsigned char* allowed, long allowed_row, const float* entropy, const float* stats, const long long* top_ids,
                                   const float* g_logprobs, long g_logprobs_stride, const float* g_entropy, long g_entropy_stride, const float* g_top,
                                   void* grad, long grad_row, long rows, int V, int top_k, int dtype, void* stream) {
  const char* who = "m2_token_scores_bwd";
  if (int rc = check_rows(who, logits, inner, outer_stride, row_stride, allowed, allowed_row, rows, V, top_k, dtype)) return rc;
  if (!entropy || !stats || !grad || (g_top && (!top_ids || !top_k)) || (g_logprobs && !tokens)) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  if (g_logprobs_stride < 0 || g_entropy_stride < 0) return set_error(M2_ERR_ARG, "%s: strides %ld and %ld", who, g_logprobs_stride, g_entropy_stride);
  if (grad_row < V) return set_error(M2_ERR_ARG, "%s: grad_row=%ld is less than V=%d", who, grad_row, V);
  if ((uintptr_t)grad % (dtype == M2_DTYPE_F32 ? 4 : 2)) return set_error(M2_ERR_UNSUPPORTED, "%s: grad must be aligned to its type", who);
  const LogitRows in = {logits, outer_stride, row_stride, inner, allowed, allowed_row};
  const ScoreGrads g = {g_logprobs, g_entropy, g_top, g_logprobs_stride, g_entropy_stride};
  hipStream_t st = (hipStream_t)stream;
  const int each = dtype == M2_DTYPE_F32 ? 4 : 8, span = 256 * kBwdChunk * each;
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((V + span - 1) / span), (unsigned)(rows < 65535 ? rows : 65535)), dim3(256), 0, st, in, tokens, ignore_index, entropy, stats, top_ids, g,
                       (char*)grad, grad_row, rows, V, top_k);
  };
  if (dtype == M2_DTYPE_F32) allowed ? go(token_scores_grad_kernel<float, true>) : go(token_scores_grad_kernel<float, false>);
  else allowed ? go(token_scores_grad_kernel<uint16_t, true>) : go(token_scores_grad_kernel<uint16_t, false>);
  return check_launch("token_scores_grad");
}
