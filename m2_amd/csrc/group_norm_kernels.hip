// Group norm with an activation on hidden states whose channels lie last, and its gradient.
//
//   a sample's group: S positions times Cg channels     m = mean x     r = 1 / sqrt(mean (x - m)^2 + eps)     xh = (x - m) r     pre = xh w + b     y = act(pre)
//   g = gy act'(pre)     t = g w     gx = r (t - mean t - xh mean(t xh))     gw = sum g xh     gb = sum g
//
// One position (groups of a token): P neighbouring lanes hold a group in registers, read once, up to 256 of the vectors that a lane moves (16 bytes where a group's channels and all addresses are
// multiples of it, else two values or one).  Wider groups of one position go with those of several, whose threads then mostly have nothing to do: 8192 x 1024 fp32 in one group with SiLU 22 us (74 with
// the gradient), 8192 x 1536 fp32 147 (447), 8192 x 3584 bf16 470 (1490), 8192 x 1002 bf16 in ones 182 (431).  Several: the values are read twice, first for means and squared distances
// of small blocks, joined with what their means differ by, so that nothing cancels; second for the result.
//
// Bound by memory: 32768 x 1536 bf16 in 24 groups with SiLU 51 us (3.9 TB/s).  8 x 2048 x 1536 with its gradient 107 us: x twice, gy and x twice more, 0.4 GB of reads and writes at 3.8 TB/s, part of
// them from the last cache; 3 x 4001 x 960 fp32 29 us (blocks 9, their join 3.6, the result 17).  Chunks that give two workgroups a compute unit: with eight, partial results and their sums took 175 us
// instead of 115.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "lane_ops.h"

namespace m2 {

struct NormArgs {
  const void *x, *gy;
  long x_sample, x_row, gy_sample, gy_row;
  const float *w, *b;      // (C) or null
  void *y, *gx;
  float* stats;            // (N, G, 2): mean, rstd
  float* partials;
  float2* sums;            // (N, G): mean t, mean t xh
  long N;
  int S, C, G, Cg, act;
  float eps;
  int columns, chunk, chunks;      // vectors of channels; positions of a chunk, chunks of a sample
};

constexpr int kSilu = 1, kGelu = 2;

template <typename T>
__device__ __forceinline__ float activate(float v, int act) {
  if (act == kSilu) return silu<T>(v);
  if (act == kGelu) return 0.5f * v * (1.f + erff(v * 0.70710678118654752440f));
  return v;
}
template <typename T>
__device__ __forceinline__ float slope(float v, int act) {
  if (act == kSilu) return silu_slope<T>(v);
  if (act == kGelu) return fmaf(v * 0.39894228040143267794f, exp_of(-0.5f * v * v), 0.5f * (1.f + erff(v * 0.70710678118654752440f)));
  return 1.f;
}

// The part of groups and rows that a lane of the one-position kernels has: NV vectors of V channels, P * V apart.
template <int V, int P, int NV>
struct Lane {
  int li, g;
  bool on;
  __device__ __forceinline__ Lane(const NormArgs& p) {
    const int lane = threadIdx.x & 63;
    li = lane % P;
    g = blockIdx.y * (64 / P) + lane / P;
    on = g < p.G;
    if (!on) g = p.G - 1;
  }
  __device__ __forceinline__ int at(int k) const { return (li + P * k) * V; }      // within the group
  __device__ __forceinline__ void weights(const NormArgs& p, float (&w)[NV][V], float (&b)[NV][V]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool in = at(k) < p.Cg;
        w[k][v] = p.w && in ? p.w[g * p.Cg + at(k) + v] : 1.f;
        b[k][v] = p.b && in ? p.b[g * p.Cg + at(k) + v] : 0.f;
      }
  }
};

template <typename T, int V, int P, int NV>
__global__ __launch_bounds__(256) void norm_rows_kernel(NormArgs p) {
  const Lane<V, P, NV> my(p);
  const int lane = threadIdx.x & 63;
  const float each = 1.f / (float)p.Cg;
  float w[NV][V], b[NV][V];
  my.weights(p, w, b);
  constexpr int U = NV == 1 ? 2 : 1;      // rows asked for together
  for (long r0 = blockIdx.x * 4L + (threadIdx.x >> 6); r0 < p.N; r0 += gridDim.x * 4L * U) {
    float f[U][NV][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long r = min(r0 + u * gridDim.x * 4L, p.N - 1);
      const T* x = static_cast<const T*>(p.x) + r * p.x_sample + my.g * p.Cg;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int v = 0; v < V; ++v) f[u][k][v] = 0.f;
        if (my.at(k) < p.Cg) load_values<T, V>(x + my.at(k), f[u][k]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long r = r0 + u * gridDim.x * 4L;
      float sum = 0.f, sq = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) sum += f[u][k][v];
      const float mean = lane_sum<P>(sum, lane) * each;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          f[u][k][v] -= mean;
          sq = fmaf(f[u][k][v], my.at(k) < p.Cg ? f[u][k][v] : 0.f, sq);
        }
      const float rstd = rsqrtf(fmaf(lane_sum<P>(sq, lane), each, p.eps));
      if (!my.on || r >= p.N) continue;
      if (my.li == 0 && p.stats) {
        p.stats[(r * p.G + my.g) * 2] = mean;
        p.stats[(r * p.G + my.g) * 2 + 1] = rstd;
      }
      T* y = static_cast<T*>(p.y) + r * p.C + my.g * p.Cg;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int v = 0; v < V; ++v) f[u][k][v] = activate<T>(fmaf(f[u][k][v] * rstd, w[k][v], b[k][v]), p.act);
        if (my.at(k) < p.Cg) store_values<T, V>(y + my.at(k), f[u][k]);
      }
    }
  }
}

template <typename T, int V, int P, int NV>
__global__ __launch_bounds__(256) void norm_rows_bwd_kernel(NormArgs p) {
  __shared__ float joined[3][64][2 * NV * V + 1];
  const Lane<V, P, NV> my(p);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float each = 1.f / (float)p.Cg;
  float w[NV][V], b[NV][V], gw[NV][V], gb[NV][V];
  my.weights(p, w, b);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) gw[k][v] = gb[k][v] = 0.f;
  for (long r = blockIdx.x * 4L + wave; r < p.N; r += gridDim.x * 4L) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_sample + my.g * p.Cg;
    const T* gy = static_cast<const T*>(p.gy) + r * p.gy_sample + my.g * p.Cg;
    const float mean = p.stats[(r * p.G + my.g) * 2], rstd = p.stats[(r * p.G + my.g) * 2 + 1];
    float xh[NV][V], t[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) xh[k][v] = mean, t[k][v] = 0.f;
      if (my.at(k) < p.Cg) {
        load_values<T, V>(x + my.at(k), xh[k]);
        load_values<T, V>(gy + my.at(k), t[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        xh[k][v] = (xh[k][v] - mean) * rstd;
        const float g = p.act ? t[k][v] * slope<T>(fmaf(xh[k][v], w[k][v], b[k][v]), p.act) : t[k][v];
        gb[k][v] += g;
        gw[k][v] = fmaf(g, xh[k][v], gw[k][v]);
        t[k][v] = g * w[k][v];
        if (my.at(k) < p.Cg) s1 += t[k][v], s2 = fmaf(t[k][v], xh[k][v], s2);
      }
    s1 = lane_sum<P>(s1, lane) * each;
    s2 = lane_sum<P>(s2, lane) * each;
    if (!my.on || !p.gx) continue;
    T* gx = static_cast<T*>(p.gx) + r * p.C + my.g * p.Cg;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) t[k][v] = rstd * (t[k][v] - fmaf(xh[k][v], s2, s1));
      if (my.at(k) < p.Cg) store_values<T, V>(gx + my.at(k), t[k]);
    }
  }
  if (!p.partials) return;
  if (wave > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) joined[wave - 1][lane][2 * (k * V + v)] = gw[k][v], joined[wave - 1][lane][2 * (k * V + v) + 1] = gb[k][v];
  }
  __syncthreads();
  if (wave > 0 || !my.on) return;
  float* out = p.partials + blockIdx.x * 2L * p.C + my.g * p.Cg;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (my.at(k) >= p.Cg) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int o = 0; o < 3; ++o) gw[k][v] += joined[o][lane][2 * (k * V + v)], gb[k][v] += joined[o][lane][2 * (k * V + v) + 1];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) out[my.at(k) + v] = gw[k][v], out[p.C + my.at(k) + v] = gb[k][v];
  }
}

// Where a thread of the kernels over many positions is: a column of V channels, and every parts-th position of a chunk.
template <int V>
struct Place {
  int lane, part, parts, column, c, g, s0, s1;
  long n;
  int chunk;
  bool on;
  __device__ __forceinline__ Place(const NormArgs& p, int CL) {
    lane = threadIdx.x % CL, part = threadIdx.x / CL, parts = 256 / CL;
    column = blockIdx.y * CL + lane;
    on = column < p.columns;
    c = on ? column * V : 0;
    g = c / p.Cg;
    n = blockIdx.x / (uint32_t)p.chunks;
    chunk = blockIdx.x - (uint32_t)n * (uint32_t)p.chunks;
    s0 = chunk * p.chunk, s1 = min(s0 + p.chunk, p.S);
  }
};

// Mean and sum of squared distances of `count` values joined into those of `total` others.
__device__ __forceinline__ void join(float& mean, float& m2, float total, float other_mean, float other_m2, float count) {
  const float d = other_mean - mean, share = count / (total + count);
  mean = fmaf(d, share, mean);
  m2 += fmaf(d, d * (total * share), other_m2);      // (a first block's d is its mean, whose square may pass fp32's range; total is 0 there)
}

template <typename T, int V>
__global__ __launch_bounds__(256) void norm_partials_kernel(NormArgs p, int CL) {
  constexpr int U = 4;
  __shared__ float2 found[256];
  __shared__ float counts[256];
  const Place<V> my(p, CL);
  const T* x = static_cast<const T*>(p.x) + my.n * p.x_sample + my.c;
  float mean = 0.f, m2 = 0.f, total = 0.f;
  for (int s = my.s0 + my.part; my.on && s < my.s1; s += U * my.parts) {
    float f[U][V], sum = 0.f, sq = 0.f;
    const int rows = min(U, (my.s1 - s + my.parts - 1) / my.parts);
#pragma unroll
    for (int u = 0; u < U; ++u) load_values<T, V>(x + min(s + u * my.parts, my.s1 - 1) * p.x_row, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < V; ++v) sum += u < rows ? f[u][v] : 0.f;
    const float count = (float)(rows * V), m = sum / count;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = f[u][v] - m;
        sq = fmaf(d, u < rows ? d : 0.f, sq);
      }
    join(mean, m2, total, m, sq, count);
    total += count;
  }
  found[threadIdx.x] = {mean, m2};
  counts[threadIdx.x] = total;
  __syncthreads();
  if (my.part > 0 || !my.on) return;
  for (int o = 1; o < my.parts; ++o) {
    const float2 f = found[o * CL + my.lane];
    const float count = counts[o * CL + my.lane];
    if (count > 0.f) join(mean, m2, total, f.x, f.y, count), total += count;
  }
  reinterpret_cast<float2*>(p.partials)[(long)blockIdx.x * p.columns + my.column] = {mean, m2};
}

__device__ __forceinline__ float block_sum(float v, float* room) {      // of 256 threads; room for 4
  const int lane = threadIdx.x & 63;
  v = lane_sum<64>(v, lane);
  __syncthreads();
  if (lane == 0) room[threadIdx.x >> 6] = v;
  __syncthreads();
  return (room[0] + room[1]) + (room[2] + room[3]);
}

// One sample's group a workgroup.
__global__ __launch_bounds__(256) void norm_stats_kernel(NormArgs p, int V) {
  __shared__ float room[4];
  const long n = blockIdx.x / (uint32_t)p.G;
  const int g = blockIdx.x - (uint32_t)n * (uint32_t)p.G, per = p.Cg / V, entries = p.chunks * per;
  const float2* found = reinterpret_cast<const float2*>(p.partials) + n * p.chunks * p.columns + g * per;
  const float all = (float)p.S * (float)p.Cg;
  float sum = 0.f, sq = 0.f;
  for (int i = threadIdx.x; i < entries; i += 256) {
    const int chunk = i / per, rows = min(p.chunk, p.S - chunk * p.chunk);
    sum = fmaf(found[(long)chunk * p.columns + i - chunk * per].x, (float)(rows * V) / all, sum);
  }
  const float mean = block_sum(sum, room);
  for (int i = threadIdx.x; i < entries; i += 256) {
    const int chunk = i / per, rows = min(p.chunk, p.S - chunk * p.chunk);
    const float2 f = found[(long)chunk * p.columns + i - chunk * per];
    const float d = f.x - mean;
    sq += fmaf(d * d, (float)(rows * V), f.y);
  }
  sq = block_sum(sq, room);
  if (threadIdx.x == 0) {
    p.stats[blockIdx.x * 2L] = mean;
    p.stats[blockIdx.x * 2L + 1] = rsqrtf(sq / all + p.eps);
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormArgs p, int CL) {
  constexpr int U = 4;
  const Place<V> my(p, CL);
  if (!my.on) return;
  const float mean = p.stats[(my.n * p.G + my.g) * 2], rstd = p.stats[(my.n * p.G + my.g) * 2 + 1];
  float w[V], b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] = p.w ? p.w[my.c + v] : 1.f, b[v] = p.b ? p.b[my.c + v] : 0.f;
  const T* x = static_cast<const T*>(p.x) + my.n * p.x_sample + my.c;
  T* y = static_cast<T*>(p.y) + my.n * p.S * p.C + my.c;
  for (int s = my.s0 + my.part; s < my.s1; s += U * my.parts) {
    float f[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_values<T, V>(x + min(s + u * my.parts, my.s1 - 1) * p.x_row, f[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int v = 0; v < V; ++v) f[u][v] = activate<T>(fmaf((f[u][v] - mean) * rstd, w[v], b[v]), p.act);
      if (s + u * my.parts < my.s1) store_values<T, V>(y + (long)(s + u * my.parts) * p.C, f[u]);
    }
  }
}

// Sums over a chunk's positions of g xh and g of every channel: (N * chunks, 2, C).
template <typename T, int V>
__global__ __launch_bounds__(256) void norm_bwd_partials_kernel(NormArgs p, int CL) {
  constexpr int U = 2;
  __shared__ float joined[256][2 * V + 1];
  const Place<V> my(p, CL);
  float gw[V], gb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) gw[v] = gb[v] = 0.f;
  if (my.on) {
    const float mean = p.stats[(my.n * p.G + my.g) * 2], rstd = p.stats[(my.n * p.G + my.g) * 2 + 1];
    float w[V], b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = p.w ? p.w[my.c + v] : 1.f, b[v] = p.b ? p.b[my.c + v] : 0.f;
    const T* x = static_cast<const T*>(p.x) + my.n * p.x_sample + my.c;
    const T* gy = static_cast<const T*>(p.gy) + my.n * p.gy_sample + my.c;
    for (int s = my.s0 + my.part; s < my.s1; s += U * my.parts) {
      float f[U][V], g[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long at = min(s + u * my.parts, my.s1 - 1);
        load_values<T, V>(x + at * p.x_row, f[u]);
        load_values<T, V>(gy + at * p.gy_row, g[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u * my.parts >= my.s1) break;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xh = (f[u][v] - mean) * rstd;
          const float d = p.act ? g[u][v] * slope<T>(fmaf(xh, w[v], b[v]), p.act) : g[u][v];
          gb[v] += d;
          gw[v] = fmaf(d, xh, gw[v]);
        }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) joined[threadIdx.x][2 * v] = gw[v], joined[threadIdx.x][2 * v + 1] = gb[v];
  __syncthreads();
  if (my.part > 0 || !my.on) return;
  float* out = p.partials + (long)blockIdx.x * 2 * p.C + my.c;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    for (int o = 1; o < my.parts; ++o) gw[v] += joined[o * CL + my.lane][2 * v], gb[v] += joined[o * CL + my.lane][2 * v + 1];
    out[v] = gw[v];
    out[p.C + v] = gb[v];
  }
}

__global__ __launch_bounds__(256) void norm_bwd_sums_kernel(NormArgs p) {
  __shared__ float room[4];
  const long n = blockIdx.x / (uint32_t)p.G;
  const int g = blockIdx.x - (uint32_t)n * (uint32_t)p.G;
  float s1 = 0.f, s2 = 0.f;
  for (long i = threadIdx.x; i < (long)p.chunks * p.Cg; i += 256) {
    const long chunk = i / p.Cg;
    const int c = g * p.Cg + (int)(i - chunk * p.Cg);
    const float* found = p.partials + (n * p.chunks + chunk) * 2 * p.C + c;
    const float w = p.w ? p.w[c] : 1.f;
    s2 = fmaf(w, found[0], s2);
    s1 = fmaf(w, found[p.C], s1);
  }
  s1 = block_sum(s1, room);
  s2 = block_sum(s2, room);
  const float all = (float)p.S * (float)p.Cg;
  if (threadIdx.x == 0) p.sums[blockIdx.x] = {s1 / all, s2 / all};
}

template <typename T, int V>
__global__ __launch_bounds__(256) void norm_bwd_apply_kernel(NormArgs p, int CL) {
  constexpr int U = 2;
  const Place<V> my(p, CL);
  if (!my.on) return;
  const float mean = p.stats[(my.n * p.G + my.g) * 2], rstd = p.stats[(my.n * p.G + my.g) * 2 + 1];
  const float2 sums = p.sums[my.n * p.G + my.g];
  float w[V], b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] = p.w ? p.w[my.c + v] : 1.f, b[v] = p.b ? p.b[my.c + v] : 0.f;
  const T* x = static_cast<const T*>(p.x) + my.n * p.x_sample + my.c;
  const T* gy = static_cast<const T*>(p.gy) + my.n * p.gy_sample + my.c;
  T* gx = static_cast<T*>(p.gx) + my.n * p.S * p.C + my.c;
  for (int s = my.s0 + my.part; s < my.s1; s += U * my.parts) {
    float f[U][V], g[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long at = min(s + u * my.parts, my.s1 - 1);
      load_values<T, V>(x + at * p.x_row, f[u]);
      load_values<T, V>(gy + at * p.gy_row, g[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xh = (f[u][v] - mean) * rstd;
        const float d = p.act ? g[u][v] * slope<T>(fmaf(xh, w[v], b[v]), p.act) : g[u][v];
        f[u][v] = rstd * (fmaf(d, w[v], -sums.x) - xh * sums.y);
      }
      if (s + u * my.parts < my.s1) store_values<T, V>(gx + (long)(s + u * my.parts) * p.C, f[u]);
    }
  }
}

namespace {

// How a call is spread.  P > 0: one position, P lanes times NV vectors a group, `blocks` workgroups along the samples.  Else chunks of positions.
struct NormPlan {
  int V, P, NV, CL, chunk, chunks;
  long blocks;
};

NormPlan norm_plan(long N, int S, int C, int G, int V) {
  NormPlan r{};
  const int Cg = C / G, vectors = Cg / V;
  r.V = V;
  if (S == 1 && vectors <= 64 * 4) {
    r.P = 1;
    while (r.P < 64 && r.P < vectors) r.P *= 2;
    r.NV = 1;
    while (r.P * r.NV < vectors) r.NV *= 2;
    const long across = (G + 64 / r.P - 1) / (64 / r.P);
    // sixteen rows a wave where that fills the chip eight times over
    r.blocks = std::max<long>((N + 63) / 64, std::min<long>((N + 3) / 4, std::max<long>(1, 8L * num_cus() / across)));
    r.blocks = std::min<long>(r.blocks, 1L << 20);
    return r;
  }
  const int columns = C / V;
  r.CL = 64;
  while (r.CL > 8 && r.CL / 2 >= columns) r.CL /= 2;
  const int parts = 256 / r.CL;
  const long across = (columns + r.CL - 1) / r.CL;
  r.chunk = 64 * parts;
  while (r.chunk > 4 * parts && N * across * ((S + r.chunk - 1) / r.chunk) < 2L * num_cus()) r.chunk /= 2;
  r.chunks = (S + r.chunk - 1) / r.chunk;
  return r;
}

int norm_vector(int C, int G, bool aligned, int dtype) {
  const int Cg = C / G, wide = dtype == M2_DTYPE_F32 ? 4 : 8;
  if (!aligned) return 1;
  if (Cg % wide == 0) return wide;
  return Cg % 2 == 0 ? 2 : 1;
}

int check_norm(const char* name, long N, int S, int C, int G, int act, int dtype) {
  if (N < 1 || S < 1 || C < 1 || G < 1 || C % G) return set_error(M2_ERR_ARG, "%s: N=%ld, S=%d, C=%d, G=%d", name, N, S, C, G);
  if (act < 0 || act > 2) return set_error(M2_ERR_ARG, "%s: activation %d", name, act);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype %d", name, dtype);
  if (C > 1 << 20 || S > 1 << 30 || N > (1L << 31) - 1 || N * G > 1L << 31 || N * S > (1L << 36) / C)
    return set_error(M2_ERR_ARG, "%s: at most 2^20 channels, 2^30 positions, 2^31 groups and 2^36 values", name);
  return M2_OK;
}

// (a grid holds below 2^32 threads)
int check_plan(const char* name, const NormPlan& plan, long N, int G) {
  if (!plan.P && (N * plan.chunks >= 1L << 24 || N * G >= 1L << 24)) return set_error(M2_ERR_ARG, "%s: N=%ld samples of several positions are more than a launch holds", name, N);
  return M2_OK;
}

bool rows_aligned(const void* p, long sample, long row, int dtype) {
  const long size = dtype == M2_DTYPE_F32 ? 4 : 2;
  return (((uintptr_t)p | (uintptr_t)(sample * size) | (uintptr_t)(row * size)) & 15) == 0;
}

// f(T, V) for what a call moves at a time
template <typename F>
void with_values(int dtype, int V, F&& f) {
  const auto types = [&](auto t) {
    using T = decltype(t);
    constexpr int wide = 16 / sizeof(T);
    if (V == wide) f(t, std::integral_constant<int, wide>{});
    else if (V == 2) f(t, std::integral_constant<int, 2>{});
    else f(t, std::integral_constant<int, 1>{});
  };
  if (dtype == M2_DTYPE_F32) types(float{});
  else types(uint16_t{});
}
template <typename F>
void with_lanes(int P, int NV, F&& f) {
  const auto vectors = [&](auto lanes) {
    if constexpr (decltype(lanes)::value == 64) {
      switch (NV) {
        case 1: return f(lanes, std::integral_constant<int, 1>{});
        case 2: return f(lanes, std::integral_constant<int, 2>{});
        default: return f(lanes, std::integral_constant<int, 4>{});
      }
    } else {
      f(lanes, std::integral_constant<int, 1>{});
    }
  };
  switch (P) {
    case 1: return vectors(std::integral_constant<int, 1>{});
    case 2: return vectors(std::integral_constant<int, 2>{});
    case 4: return vectors(std::integral_constant<int, 4>{});
    case 8: return vectors(std::integral_constant<int, 8>{});
    case 16: return vectors(std::integral_constant<int, 16>{});
    case 32: return vectors(std::integral_constant<int, 32>{});
    default: return vectors(std::integral_constant<int, 64>{});
  }
}

// Bytes of partial results: of the forward (means and squared distances), or of the gradient with the sums of groups behind them.
size_t norm_bytes(long N, int S, int C, int G, int V, bool backward) {
  const NormPlan r = norm_plan(N, S, C, G, V);
  if (r.P) return backward ? sizeof(float) * 2 * (size_t)r.blocks * C : 0;
  if (!backward) return sizeof(float2) * (size_t)N * r.chunks * (C / V);
  return sizeof(float2) * ((size_t)N * r.chunks * C + (size_t)N * G);
}

}  // namespace
}  // namespace m2

using namespace m2;

extern "C" size_t m2_group_norm_workspace_bytes(long N, int S, int C, int G, int backward, int dtype) {
  if (check_norm("group_norm", N, S, C, G, 0, dtype)) return 0;
  size_t most = 0;      // whatever the alignment
  for (bool aligned : {false, true}) most = std::max(most, norm_bytes(N, S, C, G, norm_vector(C, G, aligned, dtype), backward));
  return most;
}

extern "C" int m2_group_norm_fwd(const void* x, long x_sample, long x_row, const float* w, const float* b, float eps, void* y, float* stats, void* workspace, long N, int S,
                                 int C, int G, int act, int dtype, void* stream) {
  if (!x || !y || !stats) return set_error(M2_ERR_ARG, "group_norm_fwd: null pointer");
  if (int rc = check_norm("group_norm_fwd", N, S, C, G, act, dtype)) return rc;
  const int V = norm_vector(C, G, rows_aligned(x, x_sample, x_row, dtype) && rows_aligned(y, 0, C, dtype), dtype);
  const NormPlan plan = norm_plan(N, S, C, G, V);
  if (!plan.P && !workspace) return set_error(M2_ERR_ARG, "group_norm_fwd: no workspace");
  if (int rc = check_plan("group_norm_fwd", plan, N, G)) return rc;
  NormArgs p{};
  p.x = x, p.x_sample = x_sample, p.x_row = x_row, p.w = w, p.b = b, p.y = y, p.stats = stats, p.partials = static_cast<float*>(workspace);
  p.N = N, p.S = S, p.C = C, p.G = G, p.Cg = C / G, p.act = act, p.eps = eps, p.columns = C / V, p.chunk = plan.chunk, p.chunks = plan.chunks;
  hipStream_t s = (hipStream_t)stream;
  with_values(dtype, V, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int W = decltype(v)::value;
    if (plan.P) {
      with_lanes(plan.P, plan.NV, [&](auto lanes, auto vectors) {
        constexpr int P = decltype(lanes)::value;
        hipLaunchKernelGGL((norm_rows_kernel<T, W, P, decltype(vectors)::value>), dim3((unsigned)plan.blocks, (G + 64 / P - 1) / (64 / P)), dim3(256), 0, s, p);
      });
      return;
    }
    const dim3 grid((unsigned)(N * plan.chunks), (p.columns + plan.CL - 1) / plan.CL);
    hipLaunchKernelGGL((norm_partials_kernel<T, W>), grid, dim3(256), 0, s, p, plan.CL);
    hipLaunchKernelGGL(norm_stats_kernel, dim3((unsigned)(N * G)), dim3(256), 0, s, p, V);
    hipLaunchKernelGGL((norm_apply_kernel<T, W>), grid, dim3(256), 0, s, p, plan.CL);
  });
  return check_launch("group_norm_fwd");
}

extern "C" int m2_group_norm_bwd(const void* x, long x_sample, long x_row, const float* w, const float* b, const float* stats, const void* gy, long gy_sample, long gy_row,
                                 void* gx, float* gw, float* gb, void* workspace, long N, int S, int C, int G, int act, int dtype, void* stream) {
  if (!x || !stats || !gy) return set_error(M2_ERR_ARG, "group_norm_bwd: null pointer");
  if (int rc = check_norm("group_norm_bwd", N, S, C, G, act, dtype)) return rc;
  const bool aligned = rows_aligned(x, x_sample, x_row, dtype) && rows_aligned(gy, gy_sample, gy_row, dtype) && rows_aligned(gx, 0, C, dtype);
  const int V = norm_vector(C, G, aligned, dtype);
  const NormPlan plan = norm_plan(N, S, C, G, V);
  if ((!plan.P || gw || gb) && !workspace) return set_error(M2_ERR_ARG, "group_norm_bwd: no workspace");
  if (int rc = check_plan("group_norm_bwd", plan, N, G)) return rc;
  NormArgs p{};
  p.x = x, p.x_sample = x_sample, p.x_row = x_row, p.gy = gy, p.gy_sample = gy_sample, p.gy_row = gy_row, p.w = w, p.b = b, p.gx = gx;
  p.stats = const_cast<float*>(stats);
  p.N = N, p.S = S, p.C = C, p.G = G, p.Cg = C / G, p.act = act, p.columns = C / V, p.chunk = plan.chunk, p.chunks = plan.chunks;
  hipStream_t s = (hipStream_t)stream;
  const long rows = plan.P ? plan.blocks : N * plan.chunks;
  p.partials = plan.P && !gw && !gb ? nullptr : static_cast<float*>(workspace);
  if (!plan.P) p.sums = reinterpret_cast<float2*>(p.partials + 2 * rows * C);
  with_values(dtype, V, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int W = decltype(v)::value;
    if (plan.P) {
      with_lanes(plan.P, plan.NV, [&](auto lanes, auto vectors) {
        constexpr int P = decltype(lanes)::value;
        hipLaunchKernelGGL((norm_rows_bwd_kernel<T, W, P, decltype(vectors)::value>), dim3((unsigned)plan.blocks, (G + 64 / P - 1) / (64 / P)), dim3(256), 0, s, p);
      });
      return;
    }
    const dim3 grid((unsigned)(N * plan.chunks), (p.columns + plan.CL - 1) / plan.CL);
    hipLaunchKernelGGL((norm_bwd_partials_kernel<T, W>), grid, dim3(256), 0, s, p, plan.CL);
    if (gx) {
      hipLaunchKernelGGL(norm_bwd_sums_kernel, dim3((unsigned)(N * G)), dim3(256), 0, s, p);
      hipLaunchKernelGGL((norm_bwd_apply_kernel<T, W>), grid, dim3(256), 0, s, p, plan.CL);
    }
  });
  if (int rc = check_launch("group_norm_bwd")) return rc;
  return gw || gb ? sum_partials(p.partials, rows, 1, C, gw, gb, s) : M2_OK;
}
