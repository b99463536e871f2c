// What a masked-LM head's logits say about given tokens: log probability, entropy, the most likely alternatives, and the gradient of the three.
//
//   z_j = x_j where token j is allowed, -inf elsewhere     m = max z     s = sum exp(z_j - m)     lp_j = z_j - m - log s     p_j = exp(lp_j)
//   H = -sum p_j lp_j = log s - sum exp(z_j - m) (z_j - m) / s
//   dx_j = sum over the outputs of g ([j is its token] - p_j) - g_H p_j (lp_j + H), 0 where z_j = -inf
//
// One pass over a row: every thread keeps the largest value it has met and both sums relative to it, and rescales them when a larger one comes.
// The largest value itself, and differences to it, are kept (and not products with log2 e, which overflow for a mask of the type's lowest value).
//
// Many rows are bound by memory and, in bf16, by nine vector instructions a value, one of them exp at four times the cost of others, nearly as much: 8192 x 30522 bf16 91 us =
// 5.5 TB/s with the vector unit busy 93 % of the cycles; 4915 x 30528 fp32 104 us = 5.8 TB/s, bf16 59 us = 5.1 TB/s, with ten alternatives 65, with 32 70; the gradient 95 us =
// 6.3 TB/s of reads and writes (its reads are partly what the pass before has left in the last cache).  Few rows by latency: 1 x 30522 6.1 us, with five alternatives
// 7.8 (a pass over the row 1.4 us, the sums of all threads 1.4, the bound of the alternatives 0.7, their vectors 1.0, their order 0.5); 615 rows, 2.4 for each
// compute unit, 12 and with ten alternatives 16 us where memory would take 7.1.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "m2_internal.h"

namespace m2 {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxTop = 32;
constexpr long kMaxGrid = 1 << 21;      // workgroups of a launch (a grid holds below 2^32 threads)
constexpr float kNegInf = -__builtin_inff();

// The rows of logits: row r starts (r / inner) * outer + (r % inner) * row values behind the first (inner 0: all rows are one group).
struct LogitRows {
  const void* x;
  long outer, row;
  uint32_t inner;
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
};

template <typename T>
__device__ __forceinline__ const char* row_of(const LogitRows& in, uint32_t r) {
  const uint32_t group = in.inner ? r / in.inner : 0, at = in.inner ? r % in.inner : r;
  return reinterpret_cast<const char*>(in.x) + (group * in.outer + at * in.row) * (long)sizeof(T);
}

// Vector i of a row and what is allowed of it.  Its offset is below 2^32 (V <= 2^30), which lets the row's address stay in scalar registers.
template <typename T, bool MASK>
struct Vector {
  u32x4_any x;
  u32x2_any a;
  __device__ __forceinline__ void load(const char* row, const unsigned char* allowed, int i) {
    x = *reinterpret_cast<const u32x4_any*>(row + (uint32_t)i * 16u);
    if (MASK) {
      const unsigned char* p = allowed + (uint32_t)i * (uint32_t)Row<T>::N;
      if (Row<T>::N == 8) a = *reinterpret_cast<const u32x2_any*>(p); else a.x = *reinterpret_cast<const u32_any*>(p);
    }
  }
  __device__ __forceinline__ void values(float (&z)[Row<T>::N]) const {
    Row<T>::unpack(x, z);
    if (MASK) {
#pragma unroll
      for (int n = 0; n < Row<T>::N; ++n) z[n] = (a[n / 4] >> (8 * (n % 4))) & 0xff ? z[n] : kNegInf;
    }
  }
};

template <typename T, bool MASK>
__device__ __forceinline__ float value_at(const char* x, const unsigned char* a, long j) {
  const float v = Row<T>::one(x, j);
  return MASK && !a[j] ? kNegInf : v;
}

// The hardware's 2^x: one ulp, results below 2^-126 are 0.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// e^d for finite d, also where d log2 e has few bits behind the point: 2^p e^(d - p ln 2).
__device__ __forceinline__ float exp_(float d) {
  const float p = d * kLog2e, e = exp2_(p);
  return fmaf(e, fmaf(p, -0.693147180559945309417f, d), e);
}

// Maximum, sum of exp(z - m) in two parts and sum of exp(z - m) (z - m).  Where one token has nearly all of the probability, log s and the entropy are what
// the others add to 1: `low` keeps what the additions to s lose.
struct Sums {
  float m, s, t, low;
};
__device__ __forceinline__ Sums nothing() { return {kNegInf, 0.f, 0.f, 0.f}; }

// a.s + a.low + v
__device__ __forceinline__ void add_up(Sums& a, float v) {
  const float s = a.s + v, other = s - a.s;
  a.low += (a.s - (s - other)) + (v - other);
  a.s = s;
}

// What sums relative to `from` become relative to `to` >= from.  Differences below -1e4 stand for all that exp takes to zero, -inf and
// (-inf) - (-inf) among them, so that nothing times zero is NaN; a NaN in the sums stays one.
__device__ __forceinline__ void rescale(Sums& a, float to) {
  const float d = fmaxf(a.m - to, -1e4f), f = exp_(d);
  a.t = f * fmaf(d, a.s, a.t);
  a.s *= f;
  a.low *= f;
  a.m = to;
}

// The sums of LANES neighbours, in all of them.
template <int LANES>
__device__ __forceinline__ Sums join_lanes(Sums a) {
  float m = a.m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  rescale(a, m);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    const float s = __shfl_xor(a.s, o), t = __shfl_xor(a.t, o), low = __shfl_xor(a.low, o);
    a.t += t;
    a.low += low;
    add_up(a, s);
  }
  return a;
}

// The sum of the values, two and two.
template <int N>
__device__ __forceinline__ float sum_of(float (&e)[N]) {
#pragma unroll
  for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) e[i] += e[i + n];
  return e[0];
}

// `c`: the largest of the values.
template <int N>
__device__ __forceinline__ void add_values(Sums& a, const float (&z)[N], float c) {
  if (c > a.m) rescale(a, c);
  const float base = a.m == kNegInf ? 0.f : a.m;      // nothing but -inf (and NaN, which has to show) so far
  float e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = z[i] - base;
    e[i] = exp2_(d * kLog2e);
    a.t = fmaf(e[i], fmaxf(d, -1e4f), a.t);
  }
  add_up(a, sum_of(e));
}

// What add_values lost of values whose only largest one is m = `a.m` then, by adding the others to its 1: up to 2^-22, which is much where the rest of the row comes to little.
template <int N>
__device__ __forceinline__ float lost_beside(const float (&z)[N], float m) {
  float e[N], others = 0.f;
  bool met = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    e[i] = exp2_((z[i] - m) * kLog2e);
    others += z[i] == m && !met ? 0.f : e[i];
    met |= z[i] == m;
  }
  return others - (sum_of(e) - 1.f);
}

// (value, id) before (other, other_id): larger value first, then the lower id.
__device__ __forceinline__ bool before(float v, int id, float w, int wid) { return v > w || (v == w && id < wid); }

// The vectors [first, end) of a row, and its last V % N values where this is the last part.
struct Span {
  int first, end, tail, V;      // tail: index of the first value behind the last vector
};

// What a thread remembers of the vectors it has met: the largest value and where it was, and the largest of the other vectors.
constexpr int kTail = -1;      // in place of a vector: the value behind them
struct Met {
  float most = kNegInf, next = kNegInf;
  int at = kTail;
  __device__ __forceinline__ void see(float c, int i) {
    next = fmaxf(next, fminf(most, c));
    at = c > most ? i : at;
    most = fmaxf(most, c);
  }
};

// A number that orders as the value does (0 behind all of them, NaN apart).
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);      // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// Larger for what comes first: larger values, of equal ones the lower id.
__device__ __forceinline__ unsigned long long key_of(float v, int id) { return (unsigned long long)ordered(v) << 32 | (uint32_t)~id; }

// The k-th largest of a wave's 64 values, which have `BITS` leading bits: bit by bit, the largest number that k of them reach.
template <int BITS>
__device__ __forceinline__ float kth_largest(float v, int k) {
  const uint32_t mine = ordered(v) >> (32 - BITS);
  uint32_t at = 0;
#pragma unroll
  for (int i = BITS - 1; i >= 0; --i) {
    const uint32_t next = at | 1u << i;
    if (__builtin_popcountll(__ballot(mine >= next)) >= k) at = next;
  }
  const uint32_t u = at >> (BITS - 1) ? at ^ (1u << (BITS - 1)) : ~at;
  return __uint_as_float(u << (32 - BITS));
}

// Largest values of a part of a row, most likely first, in v and id (empty places: -inf, -1).  Called by the whole workgroup.
//
// The pass over the row leaves every thread with the largest value it has met.  Lane l of all waves is group l, of 64: the k-th largest of the groups' maxima is
// a lower bound b of the k-th largest value.  Threads that met one of at least b, k and a few in general, read its vector again, or all their vectors where the
// largest value of the others reaches b too, and what reaches b is put in order by counting.  Values equal to b may be any number (a row of one value): where they do not fit, they are taken from the front, reading in order.
// Where the values above b do not fit (all large values of a row in one group), the alternatives are looked for one after the other.
template <typename T, bool MASK, int THREADS>
struct Top {
  static constexpr int kRoom = 512, kWaves = THREADS / 64;
  float v[kMaxTop];
  int id[kMaxTop];
  float most[kWaves][64];
  unsigned long long above_key[kRoom];
  int equal_i[kRoom];
  int above, equal, chosen, count[kWaves], list[THREADS];
  float bound;

  __device__ void one_by_one(const char* x, const unsigned char* a, const Span& p, int k) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float last_v = __builtin_inff();
    int last_i = -1;
    for (int n = 0; n < k; ++n) {
      float bv = kNegInf;
      int bi = 0x7fffffff;
      const auto see = [&](int j) {
        const float z = value_at<T, MASK>(x, a, j);
        if (before(last_v, last_i, z, j) && before(z, j, bv, bi)) bv = z, bi = j;
      };
      for (int j = p.first * Row<T>::N + tid; j < p.end * Row<T>::N; j += THREADS) see(j);
      if (p.tail + tid < p.V) see(p.tail + tid);
      for (int o = 32; o > 0; o >>= 1) {
        const float ov = __shfl_xor(bv, o);
        const int oi = __shfl_xor(bi, o);
        if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
      }
      if (lane == 0) most[0][wave] = bv, count[wave] = bi;
      __syncthreads();
      for (int w = 0; w < kWaves; ++w)
        if (before(most[0][w], count[w], bv, bi)) bv = most[0][w], bi = count[w];
      __syncthreads();
      if (tid == 0) v[n] = bv, id[n] = bv == kNegInf ? -1 : bi;
      last_v = bv;
      last_i = bi;
    }
    __syncthreads();
  }

  // The first `want` places that hold `b`, which there are.
  __device__ void first_equal(const char* x, const unsigned char* a, const Span& p, float b, int want) {
    constexpr int N = Row<T>::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int found = 0;
    const auto take = [&](const float* z, int n, int j) {      // n values from place j on; the threads' places ascend
      int mine = 0;
      for (int i = 0; i < n; ++i) mine += z[i] == b;
      int upto = mine;
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(upto, o);
        if (lane >= o) upto += u;
      }
      if (lane == 63) count[wave] = upto;
      __syncthreads();
      int at = found + upto - mine;
      for (int w = 0; w < wave; ++w) at += count[w];
      for (int i = 0; i < n; ++i)
        if (z[i] == b) {
          if (at < kRoom) equal_i[at] = j + i;
          ++at;
        }
      for (int w = 0; w < kWaves; ++w) found += count[w];
      __syncthreads();
    };
    for (int base = p.first; base < p.end && found < want; base += THREADS) {
      float z[N] = {};
      const int i = base + tid, n = i < p.end ? N : 0;
      if (n) {
        Vector<T, MASK> q;
        q.load(x, a, i);
        q.values(z);
      }
      take(z, n, i * N);
    }
    if (found < want) {
      const bool in = p.tail + tid < p.V;
      const float z = in ? value_at<T, MASK>(x, a, p.tail + tid) : 0.f;
      take(&z, in, p.tail + tid);
    }
  }

  __device__ void find(const char* x, const unsigned char* a, const Span& p, const Met& met, int k) {
    constexpr int N = Row<T>::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    most[wave][lane] = met.most;
    if (tid < k) v[tid] = kNegInf, id[tid] = -1;
    __syncthreads();
    if (wave == 0) {
      float group = met.most;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) group = fmaxf(group, most[w][lane]);
      const float b = kth_largest<8 * (int)sizeof(T)>(group, k);
      if (lane == 0) bound = b, above = equal = chosen = 0;
    }
    __syncthreads();
    const float b = bound;
    const auto see = [&](float z, int j) {
      if (z > b) {
        const int at = atomicAdd(&above, 1);
        if (at < kRoom) above_key[at] = key_of(z, j);
      } else if (z == b && b > kNegInf) {
        const int at = atomicAdd(&equal, 1);
        if (at < kRoom) equal_i[at] = j;
      }
    };
    const auto see_vector = [&](int i) {
      Vector<T, MASK> q;
      q.load(x, a, i);
      float z[N];
      q.values(z);
      float c = z[0];
#pragma unroll
      for (int n = 1; n < N; ++n) c = fmaxf(c, z[n]);
      if (c >= b)
        for (int n = 0; n < N; ++n) see(z[n], i * N + n);
    };
    if (met.most >= b && met.most > kNegInf) {
      if (met.next >= b && met.next > kNegInf) {
        list[atomicAdd(&chosen, 1)] = tid;
        if (p.tail + tid < p.V) see(value_at<T, MASK>(x, a, p.tail + tid), p.tail + tid);
      } else if (met.at == kTail) {
        see(met.most, p.tail + tid);
      } else {
        see_vector(met.at);
      }
    }
    __syncthreads();
    // all vectors of the threads that met such values in more than one: as many threads to each as there are
    const int n = chosen;
    if (n > 0) {
      const int each = THREADS / n, sub = tid / n;
      if (sub < each)
        for (int i = p.first + list[tid - sub * n] + THREADS * sub; i < p.end; i += THREADS * each) see_vector(i);
    }
    __syncthreads();
    const int na = above;
    int ne = equal;
    __syncthreads();
    if (na > kRoom) return one_by_one(x, a, p, k);
    if (na < k && ne > kRoom) {
      first_equal(x, a, p, b, k - na);
      __syncthreads();
      ne = k - na;
    }
    for (int i = tid; i < na; i += THREADS) {
      const unsigned long long mine = above_key[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < na; ++j) rank += above_key[j] > mine;
      if (rank < k) v[rank] = unordered(mine >> 32), id[rank] = (int)~(uint32_t)mine;
    }
    if (na < k)
      for (int i = tid; i < ne; i += THREADS) {
        int rank = na;
#pragma unroll 8
        for (int j = 0; j < ne; ++j) rank += equal_i[j] < equal_i[i];
        if (rank < k) v[rank] = b, id[rank] = equal_i[i];
      }
    __syncthreads();
  }
};

// What is said of each row; see m2_amd.h.
struct RowScores {
  const long long* tokens;
  long long ignore_index;
  float *logprobs, *entropy, *stats;
  long long* top_ids;
  float* top_logprobs;
};

constexpr int kMaxParts = 32;

struct PartScores {
  Sums sums;
  float v[kMaxTop];
  int id[kMaxTop];
};

// The value at a row's token, for the first thread; NaN where there is none.  The token is asked for before the row is read, its value behind it.
template <typename T, bool MASK>
__device__ __forceinline__ float token_value(long long t, int V, const char* x, const unsigned char* a) {
  if (threadIdx.x != 0) return 0.f;
  return t < 0 || t >= V ? __builtin_nanf("") : value_at<T, MASK>(x, a, t);
}

__device__ __forceinline__ void finish(const RowScores& out, long r, int top_k, long long id_given, float token, const Sums& all, const float* v, const int* id) {
  const int tid = threadIdx.x;
  const bool empty = all.s == 0.f, broken = all.s != all.s;      // broken: a NaN or +inf among the values
  const float logs = empty ? 0.f : log1pf((all.s - 1.f) + all.low), nan = __builtin_nanf("");
  if (tid == 0) {
    if (out.tokens) {
      const float lp = broken ? nan : token == kNegInf ? kNegInf : (token - all.m) - logs;
      out.logprobs[r] = id_given == out.ignore_index ? 0.f : lp;
    }
    out.entropy[r] = empty ? 0.f : logs - all.t / all.s;
    out.stats[2 * r] = broken ? nan : all.m;
    out.stats[2 * r + 1] = logs;
  }
  if (tid < top_k) {
    const int at = broken ? -1 : id[tid];
    out.top_ids[r * top_k + tid] = at;
    out.top_logprobs[r * top_k + tid] = broken ? nan : at < 0 ? kNegInf : (v[tid] - all.m) - logs;
  }
}

// One workgroup a row, or a part of one where `parts` > 1: then what it found goes to `work` and token_scores_join_kernel puts the parts together.
template <typename T, bool MASK, bool TOP, int THREADS>
__global__ __launch_bounds__(THREADS) void token_scores_kernel(LogitRows in, RowScores out, uint32_t first, int V, int top_k, int parts, PartScores* __restrict__ work) {
  constexpr int N = Row<T>::N, kWaves = THREADS / 64, kAhead = 4;
  __shared__ Sums part_sums[kWaves];
  __shared__ Top<T, MASK, THREADS> top;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nvec = V / N, each = (nvec + parts - 1) / parts;
  const uint32_t b = first + blockIdx.x;
  const uint32_t r = parts > 1 ? b / parts : b;
  const int part = parts > 1 ? b % parts : 0;
  const long long token = out.tokens && tid == 0 ? out.tokens[r] : 0;
  const char* x = row_of<T>(in, r);
  const unsigned char* a = MASK ? in.allowed + r * in.allowed_row : nullptr;
  const Span p = {min(part * each, nvec), min((part + 1) * each, nvec), part == parts - 1 ? nvec * N : V, V};
  Sums mine = nothing();
  int i = p.first + tid;
  int peak = -1;      // where this thread's largest value was, 2 i + (whether `together`), -1 behind the vectors
  Met met;
  // kTogether vectors at a time, with one look at the maximum and one addition to the sum
  const auto add = [&](const auto* q, auto count, int at) {
    constexpr int C = decltype(count)::value;
    float z[C * N], c[C], all = kNegInf;
#pragma unroll
    for (int v = 0; v < C; ++v) {
      float (&zv)[N] = *reinterpret_cast<float (*)[N]>(z + v * N);
      q[v].values(zv);
      c[v] = zv[0];
#pragma unroll
      for (int n = 1; n < N; ++n) c[v] = fmaxf(c[v], zv[n]);
      if (TOP) met.see(c[v], at + v * THREADS);
      all = fmaxf(all, c[v]);
    }
    peak = all > mine.m ? 2 * at + (C > 1) : peak;
    add_values<C * N>(mine, z, all);
  };
  constexpr int kTogether = 16 / N;
  const std::integral_constant<int, kTogether> together;
  const std::integral_constant<int, 1> one;
  for (; i + (kAhead - 1) * THREADS < p.end; i += kAhead * THREADS) {
    Vector<T, MASK> q[kAhead];
#pragma unroll
    for (int c = 0; c < kAhead; ++c) q[c].load(x, a, i + c * THREADS);
#pragma unroll
    for (int c = 0; c < kAhead; c += kTogether) add(q + c, together, i + c * THREADS);
  }
  // the last vectors: as many loads at a time
  Vector<T, MASK> q[kAhead - 1];
#pragma unroll
  for (int c = 0; c < kAhead - 1; ++c)
    if (i + c * THREADS < p.end) q[c].load(x, a, i + c * THREADS);
#pragma unroll
  for (int c = 0; c < kAhead - 1; ++c)
    if (i + c * THREADS < p.end) add(q + c, one, i + c * THREADS);
  if (p.tail + tid < V) {
    const float z[1] = {value_at<T, MASK>(x, a, p.tail + tid)};
    if (TOP) met.see(z[0], kTail);
    peak = z[0] > mine.m ? -1 : peak;
    add_values<1>(mine, z, z[0]);
  }
  const float at_token = parts > 1 ? 0.f : token_value<T, MASK>(token, V, x, a);
  const float own = mine.m;
  mine = join_lanes<64>(mine);
  if (lane == 0) part_sums[wave] = mine;
  __syncthreads();
  Sums all = join_lanes<kWaves>(part_sums[lane % kWaves]);
  // One value has nearly all: what was lost beside it (2^-22 at most, 2^-18 of the rest where that is 1 / 16 of it) is looked up again.  The others cannot be as large.
  // 615 rows of 30528 bf16, ten alternatives: 16.0 -> 16.6 us.  Entropies of 0.0014 were off by 4e-5 of them, by 4e-7 this way.
  if (__builtin_amdgcn_readfirstlane((all.s - 1.f) + all.low < 0.0625f && all.m > kNegInf)) {      // the first lanes of all waves have the same numbers
    __shared__ float lost;
    if (own == all.m) {
      float l = 0.f;
      if (peak >= 0) {
        float z[kTogether * N];
#pragma unroll
        for (int v = 0; v < kTogether; ++v) {
          Vector<T, MASK> w;
          float (&zv)[N] = *reinterpret_cast<float (*)[N]>(z + v * N);
          if (v == 0 || (peak & 1)) {
            w.load(x, a, (peak >> 1) + v * THREADS);
            w.values(zv);
          } else {
#pragma unroll
            for (int n = 0; n < N; ++n) zv[n] = kNegInf;
          }
        }
        l = peak & 1 ? lost_beside<kTogether * N>(z, own) : lost_beside<N>(*reinterpret_cast<float (*)[N]>(z), own);
      }
      lost = l;
    }
    __syncthreads();
    all.low += lost;
  }
  if (TOP)
    if (all.s == all.s) top.find(x, a, p, met, top_k);
  if (parts > 1) {
    PartScores& to = work[b];
    if (tid == 0) to.sums = all;
    if (TOP && tid < top_k) to.v[tid] = top.v[tid], to.id[tid] = top.id[tid];
  } else {
    finish(out, r, top_k, token, at_token, all, top.v, top.id);
  }
}

// The parts of a row, a workgroup each: the largest of all parts' largest, in order, by counting.
template <typename T, bool MASK>
__global__ __launch_bounds__(256) void token_scores_join_kernel(LogitRows in, RowScores out, int V, int top_k, int parts, const PartScores* __restrict__ work) {
  constexpr int kTogether = 8;      // parts that are searched at the same time
  __shared__ unsigned long long key[kMaxParts * kMaxTop];
  __shared__ float best_v[kMaxTop];
  __shared__ int best_i[kMaxTop];
  const int tid = threadIdx.x;
  const uint32_t r = blockIdx.x;
  const PartScores* from = work + r * parts;
  const long long token = out.tokens && tid == 0 ? out.tokens[r] : 0;
  const Sums all = join_lanes<kMaxParts>(tid % kMaxParts < parts ? from[tid % kMaxParts].sums : nothing());
  if (top_k && all.s == all.s) {
    // larger values first, then lower ids: all keys are different, empty places are 0
    for (int i = tid; i < (parts + kTogether - 1) / kTogether * kTogether * kMaxTop; i += 256) {
      const int p = i / kMaxTop, n = i % kMaxTop;
      const bool is = p < parts && n < top_k && from[p].id[n] >= 0;
      key[i] = is ? key_of(from[p].v[n], from[p].id[n]) : 0;
    }
    if (tid < top_k) best_v[tid] = kNegInf, best_i[tid] = -1;
    __syncthreads();
    for (int i = tid; i < parts * kMaxTop; i += 256) {
      const unsigned long long mine = key[i];
      int rank = 0;
      // how many come before in each part, which is sorted
      for (int p = 0; p < parts; p += kTogether) {
        int at[kTogether] = {};
#pragma unroll
        for (int step = kMaxTop / 2; step > 0; step /= 2)
#pragma unroll
          for (int q = 0; q < kTogether; ++q) at[q] += key[(p + q) * kMaxTop + at[q] + step - 1] > mine ? step : 0;
#pragma unroll
        for (int q = 0; q < kTogether; ++q) rank += at[q] + (key[(p + q) * kMaxTop + at[q]] > mine ? 1 : 0);
      }
      if (mine && rank < top_k) best_v[rank] = unordered(mine >> 32), best_i[rank] = (int)~(uint32_t)mine;
    }
  }
  const float at_token = token_value<T, MASK>(token, V, row_of<T>(in, r), MASK ? in.allowed + r * in.allowed_row : nullptr);
  __syncthreads();
  finish(out, r, top_k, token, at_token, all, best_v, best_i);
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
                                                                long grad_row, uint32_t first_row, uint32_t chunks, int V, int top_k) {
  constexpr int N = Row<T>::N;
  __shared__ int ids[kMaxTop + 1];
  __shared__ float gs[kMaxTop + 1];
  const int tid = threadIdx.x;
  const uint32_t chunk = blockIdx.x % chunks;
  const long r = first_row + blockIdx.x / chunks;
  const char* x = row_of<T>(in, (uint32_t)r);
  const unsigned char* a = MASK ? in.allowed + r * in.allowed_row : nullptr;
  char* out = grad + r * grad_row * (long)sizeof(T);
  const int nvec = V / N, first = (int)chunk * 256 * kBwdChunk, lo = first * N;
  Vector<T, MASK> q[kBwdChunk];      // asked for before all else
#pragma unroll
  for (int c = 0; c < kBwdChunk; ++c)
    if (first + c * 256 + tid < nvec) q[c].load(x, a, first + c * 256 + tid);
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
#pragma unroll
  for (int c = 0; c < kBwdChunk; ++c) {
    const int i = first + c * 256 + tid;
    if (i < nvec) {
      float z[N];
      q[c].values(z);
#pragma unroll
      for (int n = 0; n < N; ++n) z[n] = slope(z[n]);
      *reinterpret_cast<u32x4_any*>(out + (long)i * 16) = Row<T>::pack(z);
    }
  }
  const bool last = chunk == chunks - 1;
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
}

static int check_rows(const char* who, const void* logits, int inner, long outer, long row, const unsigned char* allowed, long allowed_row, long rows,
                      int V, int top_k, int dtype) {
  if (!logits) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype must be M2_DTYPE_F32 or M2_DTYPE_BF16 (got %d)", who, dtype);
  if (rows <= 0 || V <= 0 || inner <= 0 || outer < 0 || row < 0) return set_error(M2_ERR_ARG, "%s: rows=%ld V=%d inner=%d outer=%ld row=%ld", who, rows, V, inner, outer, row);
  if (rows > 0x7fffffffL) return set_error(M2_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows (rows=%ld)", who, rows);
  if (V > (1 << 30)) return set_error(M2_ERR_UNSUPPORTED, "%s: at most 2^30 values in a row (V=%d)", who, V);
  if (top_k < 0 || top_k > kMaxTop || top_k > V) return set_error(M2_ERR_UNSUPPORTED, "%s: 0 to %d alternatives, at most V (top_k=%d V=%d)", who, kMaxTop, top_k, V);
  if (allowed && allowed_row != 0 && allowed_row < V) return set_error(M2_ERR_ARG, "%s: allowed_row=%ld is less than V=%d", who, allowed_row, V);
  if ((uintptr_t)logits % (dtype == M2_DTYPE_F32 ? 4 : 2)) return set_error(M2_ERR_UNSUPPORTED, "%s: logits must be aligned to their type", who);
  return M2_OK;
}

}  // namespace m2

using namespace m2;

// Workgroups a row: the second kernel, which puts parts together, costs 4 us, so rows of fewer than 8192 vectors stay whole, and there is no use for more parts than
// fill the chip.  us, 1 / 2 / 4 / 8 / 16 parts, 512 threads: 131072 fp32 top 32 1 row 18.1 / 16.8 / 14.0 / 13.0 / 14.9, 24 rows 18.8 / 17.4 / 14.8 / 13.7 / 16.8; 30528 bf16 top 5
// 1 row 7.7 / 10.9 / 9.4 / 9.5 / 12.0.
static int parts_of(long rows, int V, int dtype) {
  const long vectors = V / (dtype == M2_DTYPE_F32 ? 4 : 8);
  long parts = vectors / 4096;
  if (parts > 512 / rows) parts = 512 / rows;
  return parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : (int)parts;
}

extern "C" size_t m2_token_scores_workspace_bytes(long rows, int V, int dtype) {
  if (rows <= 0 || V <= 0) return 0;
  const int parts = parts_of(rows, V, dtype);
  return parts > 1 ? (size_t)rows * parts * sizeof(PartScores) : 0;
}

extern "C" int m2_token_scores_fwd(const void* logits, int inner, long outer_stride, long row_stride, const long long* tokens, long long ignore_index,
                                   const unsigned char* allowed, long allowed_row, float* logprobs, float* entropy, float* stats, long long* top_ids,
                                   float* top_logprobs, void* workspace, long rows, int V, int top_k, int dtype, void* stream) {
  const char* who = "m2_token_scores_fwd";
  if (int rc = check_rows(who, logits, inner, outer_stride, row_stride, allowed, allowed_row, rows, V, top_k, dtype)) return rc;
  if (!entropy || !stats || (tokens && !logprobs) || (top_k && (!top_ids || !top_logprobs))) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  const int parts = parts_of(rows, V, dtype);
  if (parts > 1 && (!workspace || (uintptr_t)workspace % 4)) return set_error(M2_ERR_ARG, "%s: rows=%ld V=%d need a workspace, aligned to 4 bytes", who, rows, V);
  const LogitRows in = {logits, outer_stride, row_stride, inner < rows ? (uint32_t)inner : 0, allowed, allowed_row};
  const RowScores out = {tokens, ignore_index, logprobs, entropy, stats, top_ids, top_logprobs};
  hipStream_t st = (hipStream_t)stream;
  const long blocks = rows * parts;
  const auto go = [&](auto kernel, int threads) {
    for (long first = 0; first < blocks; first += kMaxGrid)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks - first < kMaxGrid ? blocks - first : kMaxGrid)), dim3(threads), 0, st, in, out, (uint32_t)first, V, top_k, parts,
                         (PartScores*)workspace);
  };
  const auto pick = [&](auto* t, auto masked) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr bool M = decltype(masked)::value;
    // us, 512 / 256 / 128 threads a row, ten alternatives: 30528 bf16 16 rows 8.2 / 9.1 / -, 300 13.0 / 12.9 / 17.9, 4915 78 / 65 / 68; 4000 bf16 8000 rows 55 / 33 / 28; 16000
    // bf16 4000 rows 47 / 38 / 36
    const int threads = blocks <= num_cus() ? 512 : V / Row<T>::N <= 2048 && blocks > 4L * num_cus() ? 128 : 256;
    if (threads == 512) top_k ? go(token_scores_kernel<T, M, true, 512>, 512) : go(token_scores_kernel<T, M, false, 512>, 512);
    else if (threads == 256) top_k ? go(token_scores_kernel<T, M, true, 256>, 256) : go(token_scores_kernel<T, M, false, 256>, 256);
    else top_k ? go(token_scores_kernel<T, M, true, 128>, 128) : go(token_scores_kernel<T, M, false, 128>, 128);
    if (parts > 1)
      hipLaunchKernelGGL((token_scores_join_kernel<T, M>), dim3((unsigned)rows), dim3(256), 0, st, in, out, V, top_k, parts, (const PartScores*)workspace);
  };
  const auto type = [&](auto* t) { allowed ? pick(t, std::true_type{}) : pick(t, std::false_type{}); };
  dtype == M2_DTYPE_F32 ? type((float*)nullptr) : type((uint16_t*)nullptr);
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
  const LogitRows in = {logits, outer_stride, row_stride, inner < rows ? (uint32_t)inner : 0, allowed, allowed_row};
  const ScoreGrads g = {g_logprobs, g_entropy, g_top, g_logprobs_stride, g_entropy_stride};
  hipStream_t st = (hipStream_t)stream;
  const int span = 256 * kBwdChunk * (dtype == M2_DTYPE_F32 ? 4 : 8);
  const uint32_t chunks = (uint32_t)((V + (long)span - 1) / span);
  const auto go = [&](auto kernel) {
    const long most = kMaxGrid / chunks;
    for (long first = 0; first < rows; first += most)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(rows - first < most ? rows - first : most) * chunks), dim3(256), 0, st, in, tokens, ignore_index, entropy, stats, top_ids, g,
                         (char*)grad, grad_row, (uint32_t)first, chunks, V, top_k);
  };
  if (dtype == M2_DTYPE_F32) allowed ? go(token_scores_grad_kernel<float, true>) : go(token_scores_grad_kernel<float, false>);
  else allowed ? go(token_scores_grad_kernel<uint16_t, true>) : go(token_scores_grad_kernel<uint16_t, false>);
  return check_launch("token_scores_grad");
}
