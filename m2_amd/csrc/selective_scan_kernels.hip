// The selective state space scan of a mixer, and its form for one token.
//
//   d = softplus(dt + bias)     h[t, n] = exp(d[t] A[n]) h[t - 1, n] + d[t] x[t] B[t, n]     y[t] = (sum_n C[t, n] h[t, n] + D x[t]) z sigmoid(z)
//
// for every channel with states n = 0 .. N - 1 of its own, B and C shared by a group of channels.
//
// A wave holds 16 positions of 64 / NS channels: for each of its states a lane forms the 16 decays and inputs, runs over them from zero, and keeps them.  The waves
// of a workgroup lie along the positions; what each of them does to a state (a product of decays and a sum) goes through shared memory, so that every wave knows the
// state it starts with and runs over its kept decays once more, now with the right state, for the outputs.  Positions are thus worked on side by side, at one more
// operation a state than one position after another takes, and the decays' exponentials, four times as costly as the others, are formed once.
//
// Bound by vector instructions (82 % of the cycles at 4 x 8192 x 1536, shared memory 38 %): nine issue slots of a state and position (product, exponential, product, three sums) and six more for
// all else, of which the step size's softplus and the gate are half.  bf16, 16 states: 4 x 8192 x 1536 350 - 365 us over several machines, where bytes would take 79; 1 x 8192 x 1536 128 - 134 (192
// workgroups for 256 compute units); fp32, 61 states, 5 x 1013 x 1002 140, with a sequence's lengths as without: neighbouring workgroups are one sequence's and lie on one XCD, so a padded batch takes as
// long as an XCD with the longest sequences does (38 % busy then).  A loop must not wait for its prefetch: a choice between two loads, or a value that is made of a loaded register only later, made the
// compiler move registers at once (4 x 8192 x 1536 464 -> 374 us without).  Addresses are a scalar and 32 bits of a lane: in 64 bits they were a tenth of all instructions.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "selective_scan.h"

namespace m2 {

// Shapes of two states a lane whose registers leave room for three waves a SIMD.
constexpr bool three_waves(int NS, int NL) { return NL == 2 && NS > 2 && NS < 32; }

template <typename T, int NS, int NL>
__global__ __launch_bounds__(three_waves(NS, NL) ? 768 : 512) __attribute__((amdgpu_waves_per_eu(three_waves(NS, NL) ? 3 : 2))) void selective_scan_kernel(ScanArgs p) {
  using S = ScanShape<NS, NL>;
  constexpr int CW = S::CW, NP = S::NP, TT = S::TT, NT = S::NT, PITCH = S::PITCH;
  constexpr int kWave = 2 * S::TILE + (NS > 1 ? 2 * CW * PITCH : 0);      // floats
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane % CW, q = lane / CW;
  const int id = xcd_order(blockIdx.x, gridDim.x), block = id % p.blocks, g = id / p.blocks % p.G, b = id / p.blocks / p.G;
  const int count = min(CW, p.per_group - block * CW);
  const bool on = c < count;
  const int ch = g * p.per_group + block * CW + min(c, count - 1);
  const int n = scan_length(p, b), span = W * TT;
  float* Bs = lds + w * kWave;
  float* Cs = Bs + S::TILE;
  float* ds = Cs + S::TILE;
  float* xs = ds + CW * PITCH;
  float* ex = lds + W * kWave;      // (2, W, 2, 64, NL)

  float A2[NL], H[NL];      // decays in powers of two; the state ahead of the step's first position
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int at = q * NL + j;
    const bool real = on && at < p.N;
    A2[j] = real ? decay_rate(p.A[(long)ch * p.N + at]) : 0.f;
    H[j] = real && p.state ? p.state[((long)b * p.channels + ch) * p.N + at] : 0.f;
  }
  const float bias = p.dt_bias ? p.dt_bias[ch] : 0.f, skip = p.D ? p.D[ch] : 0.f;
  const T* x = static_cast<const T*>(p.x) + b * p.x_batch;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dt_batch;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_batch : x;      // (no gate: loads that nothing comes of, rather than waits around a branch)
  const long z_row = p.z ? p.z_row : p.x_row;
  const T* Bm = static_cast<const T*>(p.Bm) + b * p.b_batch + g * p.b_group;
  const T* Cm = static_cast<const T*>(p.Cm) + b * p.c_batch + g * p.c_group;
  T* y = static_cast<T*>(p.y) + (long)b * p.L * p.channels;
  // a lane moves positions q, q + NS, ... of its channel (lanes beyond the 16th of a channel none)
  const bool moves = NS <= TT || q < TT;
  const int q0 = NS <= TT ? q : min(q, TT - 1);

  const uint32_t y_off = (uint32_t)(q0 * p.channels + ch) * sizeof(T);
  T rx[NT], rdt[NT], rz[NT];
  TileIn<T, NS, NL, S::AHEAD ? S::NB : 1> rb, rc;      // where they fit into registers, a step's tiles are asked for ahead
  const auto load = [&](int t0) {
    t0 = min(t0, n - 1);      // (a wave whose positions all lie behind the end)
    const int last = min(n - 1 - t0, TT - 1);
    const Near x_off = Near::of(x, q0, p.x_row, ch, last), dt_off = Near::of(dt, q0, p.dt_row, ch, last), z_off = Near::of(z, q0, z_row, ch, last);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t t = i * NS * sizeof(T);
      rx[i] = at_offset<const T>(x + t0 * p.x_row, x_off(t * (uint32_t)p.x_row)), rdt[i] = at_offset<const T>(dt + t0 * p.dt_row, dt_off(t * (uint32_t)p.dt_row));
      rz[i] = at_offset<const T>(z + t0 * z_row, z_off(t * (uint32_t)z_row));
    }
    if constexpr (S::AHEAD) {
      rb.load(Bm, p.b_row, t0, n, p.N, lane);
      rc.load(Cm, p.c_row, t0, n, p.N, lane);
    }
  };
  const int steps = (n + span - 1) / span;
  if (steps > 0) load(w * TT);
  for (int s = 0; s < steps; ++s) {
    const int t0 = s * span + w * TT;
    float xv[NT], gate[NT], own_d[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const bool inside = t0 + q0 + i * NS < n;
      xv[i] = value_of<T>(rx[i]);
      float d = value_of<T>(rdt[i]) + bias;
      if (p.softplus) d = softplus(d);
      own_d[i] = inside ? d : 0.f;
      xv[i] = inside ? xv[i] : 0.f;
      gate[i] = p.z ? silu<T>(value_of<T>(rz[i])) : 1.f;
    }
    wave_sync();      // the tiles have been read
    if constexpr (S::AHEAD) {
      rb.put(Bs, p.N, lane);
      rc.put(Cs, p.N, lane);
    } else {
      tile_in<T, NS, NL>(Bs, Bm, p.b_row, min(t0, n - 1), n, p.N, lane);
      tile_in<T, NS, NL>(Cs, Cm, p.c_row, min(t0, n - 1), n, p.N, lane);
    }
    if constexpr (NS > 1) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (moves) ds[c * PITCH + q0 + i * NS] = own_d[i], xs[c * PITCH + q0 + i * NS] = own_d[i] * xv[i];
    }
    wave_sync();
    if (s + 1 < steps) load(t0 + span);
    float a[TT][NL], u[TT][NL], h[NL], total = 0.f;
#pragma unroll
    for (int j = 0; j < NL; ++j) h[j] = 0.f;
#pragma unroll
    for (int t4 = 0; t4 < TT; t4 += 4) {
      float d4[4], x4[4];
      if constexpr (NS > 1) {
        load_values<float, 4>(ds + c * PITCH + t4, d4);
        load_values<float, 4>(xs + c * PITCH + t4, x4);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) d4[i] = own_d[(t4 + i) % NT], x4[i] = d4[i] * xv[(t4 + i) % NT];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t4 + i;
        float bn[NL];
        load_values<float, NL>(Bs + t * NP + q * NL, bn);
        total += d4[i];
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          a[t][j] = __builtin_amdgcn_exp2f(d4[i] * A2[j]);
          u[t][j] = x4[i] * bn[j];
          h[j] = fmaf(a[t][j], h[j], u[t][j]);
        }
      }
    }
    float P[NL], start[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) P[j] = __builtin_amdgcn_exp2f(total * A2[j]), start[j] = 0.f;

    if (W == 1) {
#pragma unroll
      for (int j = 0; j < NL; ++j) start[j] = H[j], H[j] = fmaf(P[j], H[j], h[j]);
    } else {
      float* turn = ex + (s & 1) * W * 2 * 64 * NL;
      store_values<float, NL>(turn + (w * 2 * 64 + lane) * NL, P);
      store_values<float, NL>(turn + ((w * 2 + 1) * 64 + lane) * NL, h);
      __syncthreads();      // (two turns: what is written next is read behind the next barrier)
      // four at a time, since one after another would wait for shared memory each (1 x 8192 x 1536 139 -> 128 us with twelve waves, 4 x 8192 x 1536 362 -> 350 with four); with four states a lane that
      // takes too many registers (61 states, 5 x 1013 x 1002 142 -> 171)
      if constexpr (NL < 4) {
        for (int first = 0; first < W; first += 4) {
          float po[4][NL], ho[4][NL];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int o = min(first + k, W - 1);
            load_values<float, NL>(turn + (o * 2 * 64 + lane) * NL, po[k]);
            load_values<float, NL>(turn + ((o * 2 + 1) * 64 + lane) * NL, ho[k]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bool here = first + k == w, met = first + k < W;
#pragma unroll
            for (int j = 0; j < NL; ++j) {
              start[j] = here ? H[j] : start[j];
              H[j] = met ? fmaf(po[k][j], H[j], ho[k][j]) : H[j];
            }
          }
        }
      } else {
        const auto meet = [&](int o) {
          float po[NL], ho[NL];
          load_values<float, NL>(turn + (o * 2 * 64 + lane) * NL, po);
          load_values<float, NL>(turn + ((o * 2 + 1) * 64 + lane) * NL, ho);
#pragma unroll
          for (int j = 0; j < NL; ++j) H[j] = fmaf(po[j], H[j], ho[j]);
        };
        for (int o = 0; o < w; ++o) meet(o);
#pragma unroll
        for (int j = 0; j < NL; ++j) start[j] = H[j];
        for (int o = w; o < W; ++o) meet(o);
      }
    }
    if (p.saved && t0 % p.apart == 0 && t0 < n && on) {
      float* kept = p.saved + (((long)b * p.parts + t0 / p.apart) * p.channels + ch) * p.N + q * NL;
#pragma unroll
      for (int j = 0; j < NL; ++j)
        if (q * NL + j < p.N) kept[j] = start[j];
    }
    float out[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float cn[NL];
      load_values<float, NL>(Cs + t * NP + q * NL, cn);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        start[j] = fmaf(a[t][j], start[j], u[t][j]);
        sum = j == 0 ? cn[0] * start[0] : fmaf(cn[j], start[j], sum);
      }
      out[t] = sum;
    }
    share_positions<NS, log2_of(CW)>(out, lane);
    if (t0 + TT <= n) {
      if (on && moves) {
#pragma unroll
        for (int i = 0; i < NT; ++i) at_offset<T>(y + (long)(t0 + i * NS) * p.channels, y_off) = value_to<T>(fmaf(skip, xv[i], out[i]) * gate[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int t = t0 + q0 + i * NS;
        const float v = fmaf(skip, xv[i], out[i]) * gate[i];
        if (on && moves && t < p.L) y[(long)t * p.channels + ch] = value_to<T>(t < n ? v : 0.f);
      }
    }
  }
  for (int t0 = steps * span + w * TT; t0 < p.L; t0 += span)
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int t = t0 + q0 + i * NS;
      if (on && moves && t < p.L) y[(long)t * p.channels + ch] = value_to<T>(0.f);
    }
  if (p.state_out && w == 0 && on) {
#pragma unroll
    for (int j = 0; j < NL; ++j)
      if (q * NL + j < p.N) p.state_out[((long)b * p.channels + ch) * p.N + q * NL + j] = H[j];
  }
}

// One token: P lanes a channel, V states a lane at a time; a thread does so for I channels (of all sequences, 256 / P apart), whose loads it asks for together.
template <typename T, int V, int I>
__global__ __launch_bounds__(256) void selective_scan_step_kernel(ScanArgs p, int P) {
  const int lane = threadIdx.x & 63, each = 256 / P;
  const uint32_t q = threadIdx.x & (P - 1), last = (uint32_t)p.batch * (uint32_t)p.channels - 1;
  uint32_t item[I], ch[I];
  const T *Bm[I], *Cm[I];
  float xv[I], d[I], zv[I], skip[I], sum[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    item[i] = (blockIdx.x * I + i) * (uint32_t)each + threadIdx.x / P;
    const uint32_t at = min(item[i], last), b = at / (uint32_t)p.channels, g = (ch[i] = at - b * (uint32_t)p.channels) / (uint32_t)p.per_group;
    Bm[i] = static_cast<const T*>(p.Bm) + b * p.b_batch + g * p.b_group;
    Cm[i] = static_cast<const T*>(p.Cm) + b * p.c_batch + g * p.c_group;
    xv[i] = value_of<T>(static_cast<const T*>(p.x)[b * p.x_batch + ch[i]]);
    d[i] = value_of<T>(static_cast<const T*>(p.dt)[b * p.dt_batch + ch[i]]);
    zv[i] = p.z ? value_of<T>(static_cast<const T*>(p.z)[b * p.z_batch + ch[i]]) : 0.f;
    skip[i] = p.D ? p.D[ch[i]] : 0.f;
    if (p.dt_bias) d[i] += p.dt_bias[ch[i]];
    sum[i] = 0.f;
  }
  for (int n = q * V; n < p.N; n += P * V) {
    float av[I][V], hv[I][V], bv[I][V], cv[I][V];
#pragma unroll
    for (int i = 0; i < I; ++i) {
      load_values<float, V>(p.state + (long)min(item[i], last) * p.N + n, hv[i]);
      load_values<float, V>(p.A + (long)ch[i] * p.N + n, av[i]);
      if constexpr (V == 4) {
        const auto b4 = *reinterpret_cast<const typename Raw4<T>::type*>(Bm[i] + n), c4 = *reinterpret_cast<const typename Raw4<T>::type*>(Cm[i] + n);
#pragma unroll
        for (int j = 0; j < V; ++j) bv[i][j] = Raw4<T>::get(b4, j), cv[i][j] = Raw4<T>::get(c4, j);
      } else {
        bv[i][0] = value_of<T>(Bm[i][n]), cv[i][0] = value_of<T>(Cm[i][n]);
      }
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      // (the step in powers of two and not A, whose product with log2 e may pass fp32's range)
      const float step = p.softplus ? softplus(d[i]) : d[i], dx = step * xv[i], twos = step * kLog2E;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        hv[i][j] = fmaf(__builtin_amdgcn_exp2f(twos * av[i][j]), hv[i][j], dx * bv[i][j]);
        sum[i] = fmaf(cv[i][j], hv[i][j], sum[i]);
      }
      if (item[i] <= last) store_values<float, V>(p.state_out + (long)item[i] * p.N + n, hv[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < I; ++i) {
    if (P > 1) sum[i] = sum_over_bit<0>(sum[i], lane);
    if (P > 2) sum[i] = sum_over_bit<1>(sum[i], lane);
    if (P > 4) sum[i] = sum_over_bit<2>(sum[i], lane);
    if (P > 8) sum[i] = sum_over_bit<3>(sum[i], lane);
    if (P > 16) sum[i] = sum_over_bit<4>(sum[i], lane);
    if (P > 32) sum[i] = sum_over_bit<5>(sum[i], lane);
    if (item[i] <= last && q == 0) {
      float v = fmaf(skip[i], xv[i], sum[i]);
      if (p.z) v *= silu<T>(zv[i]);
      static_cast<T*>(p.y)[item[i]] = value_to<T>(v);
    }
  }
}

namespace {

constexpr int kMaxStates = 256;

int check_scan(const char* name, const ScanArgs& p, int dtype) {
  if (p.batch < 1 || p.L < 1 || p.channels < 1 || p.G < 1 || p.channels % p.G) return set_error(M2_ERR_ARG, "%s: B=%d, L=%d, D=%d, G=%d", name, p.batch, p.L, p.channels, p.G);
  if (p.N < 1 || p.N > kMaxStates) return set_error(M2_ERR_UNSUPPORTED, "%s: N=%d states, 1 .. %d are supported", name, p.N, kMaxStates);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype %d", name, dtype);
  for (long row : {p.x_row, p.dt_row, p.z_row, p.b_row, p.c_row, p.gy_row})
    if (row < 0 || row >= 1L << 24) return set_error(M2_ERR_UNSUPPORTED, "%s: rows %ld values apart, below 2^24 are supported", name, row);
  if ((long)p.batch * p.L >= (1L << 32) / ((long)p.G * p.N)) return set_error(M2_ERR_ARG, "%s: below 2^32 values of B are supported", name);
  if (p.channels > 1 << 20 || p.L > 1 << 30 || (long)p.batch * p.channels > 1L << 26)
    return set_error(M2_ERR_ARG, "%s: at most 2^20 channels, 2^30 positions and 2^26 channels of all sequences", name);
  return M2_OK;
}

int check_grid(const char* name, const ScanArgs& p, const ScanPlan& plan) {
  if ((long)plan.blocks * p.G * p.batch * plan.W >= 1L << 26) return set_error(M2_ERR_ARG, "%s: B=%d, D=%d, N=%d are more than a launch holds", name, p.batch, p.channels, p.N);
  return M2_OK;
}

int pow2_from(int n) {
  int r = 1;
  while (r < n) r *= 2;
  return r;
}

size_t fwd_lds(const ScanPlan& s) {
  const int CW = 64 / s.NS;
  return sizeof(float) * s.W * (2 * 16 * s.NS * s.NL + (s.NS > 1 ? 2 * CW * 20 : 0) + (s.W > 1 ? 2 * 2 * 64 * s.NL : 0));
}

// Lanes a channel and states a lane.  A wave's sixteen positions cost some 150 instructions for each state of a lane (a product, an exponential at four times the cost of others, a product,
// three sums), 45 for each position whose x, dt, z and y it moves, a sum across lanes, and 60 for what all waves do; four states a lane leave room for two waves a SIMD instead of
// three (8 % more).  What counts is the share of the compute unit with most workgroups.  us with four / two / one a lane, each with its best number of waves: 16 states, 1 x 8192 x 1536 218 / 128 / 161
// (96, 192, 384 workgroups), 4 x 8192 x 1536 418 / 350 / 505 (384, 768, 1536), 8 x 2048 x 1536 174 / 164 / - (the rule takes four); 61 states, 5 x 1013 x 1002 140 / 198 / 231.
template <typename SHAPES>
void choose_shape(ScanPlan& r, int B, int D, int G, int N) {
  const int per_group = D / G, cus = num_cus();
  double least = 0;
  for (int NL : {4, 2, 1}) {
    const int NS = std::max(pow2_from((N + NL - 1) / NL), SHAPES::built(1, 1) ? 1 : 2);
    if (NS > 64 || !SHAPES::built(NS, NL)) continue;
    const int CW = 64 / NS, blocks = (per_group + CW - 1) / CW;
    const long share = ((long)blocks * G * B + cus - 1) / cus;
    const double cost = (150 * NL + 45 * std::max(16 / NS, 1) + 2.5 * (16 - 16 / std::min(NS, 16)) + 60) * (NL == 4 ? 1.08 : 1.0) * share;
    if (least == 0 || cost < least) least = cost, r.NS = NS, r.NL = NL, r.blocks = blocks;
  }
}
// Waves of a workgroup: eight, or twelve with two states a lane, where a compute unit has one workgroup; fewer, down to two, where more share its registers (two or three waves a SIMD); as many as there
// are positions for.  us with two / four / eight / twelve waves and two states a lane: 1 x 8192 x 1536 (one workgroup a compute unit) 395 / 213 / 143 / 128, 4 x 8192 x 1536 (three) 499 / 350 / 438,
// 8 x 2048 x 1536 (six) 164 / 166 / 226; four states a lane with four / eight: 4 x 8192 x 1536 (two workgroups) 418 / 446, 8 x 2048 x 1536 (three) 184 / 174.
ScanPlan fwd_plan(int B, int L, int D, int G, int N) {
  ScanPlan r{};
  choose_shape<ForwardShapes>(r, B, D, G, N);
  const long share = ((long)r.blocks * G * B + num_cus() - 1) / num_cus();
  const int room = three_waves(r.NS, r.NL) ? 12 : r.NL == 1 ? 16 : 8;
  r.W = three_waves(r.NS, r.NL) && share == 1 ? 12 : 8;
  if (r.NL == 4) r.W = share % 2 ? 8 : 4;      // one workgroup at a time fills a compute unit with eight, two with four
  else while (r.W > 2 && r.W * share > room) r.W /= 2;
  while (r.W > 1 && (r.W / 2) * 16 >= L) r.W /= 2;
  while (fwd_lds(r) > (share == 1 ? 150 << 10 : 80 << 10)) r.W /= 2;
  return r;
}
// The gradient: sets of channels that a workgroup takes one after the other, so that it writes one partial gradient of B and C for all of them: as many as leave the share of
// the compute unit with most of them as it is, and three workgroups for each.  8 x 2048 x 1536 of 16 states, us with the forward: one set 815, two 724, three 759.  More where the
// partial gradients would take more than 1 GiB and sixteen bytes for each value of x (many states, whose workgroups have few channels a set), as long as each compute unit keeps a workgroup.
// The gradient alone, ms, with sets for the memory alone / as here / three of them: 1 x 16384 x 1536 of 128 states 41.8 (64 workgroups, 1 GiB) / 14.2 (256, 4) / 11.1 (512, 8);
// 1 x 8192 x 1536 of 128 11.6 (128, 1) / 7.2 (256, 2) / 5.6 (512, 4); 1 x 32768 x 768 of 64 17.4 (64, 1) / 6.6 (256, 4) / 6.6.
ScanPlan bwd_plan(int B, int L, int D, int G, int N) {
  ScanPlan r{};
  choose_shape<GradientShapes>(r, B, D, G, N);
  r.W = m2_selective_scan_span(N) / 16;      // a step from each state that is kept
  const int sets = r.blocks, cus = num_cus();
  long least = 0;
  for (int each = 1; each <= 8; ++each) {
    const ScanPlan t{r.NS, r.NL, r.W, (sets + each - 1) / each, each};
    const long groups = (long)t.blocks * G * B, share = (groups + cus - 1) / cus * each;
    if (each > 1 && (groups < 3L * cus || scan_bwd_lds(t) > (53 << 10))) break;
    if (least == 0 || share <= least) least = share, r.blocks = t.blocks, r.sets = each;
  }
  const double values = (double)B * L, most = std::max(1073741824.0, 16 * values * D);
  for (int each = r.sets + 1; each <= std::min(64, sets) && 8 * values * r.blocks * G * N > most; ++each) {
    const ScanPlan t{r.NS, r.NL, r.W, (sets + each - 1) / each, each};
    if ((long)t.blocks * G * B < cus || scan_bwd_lds(t) > (160 << 10)) break;
    r.blocks = t.blocks, r.sets = each;
  }
  return r;
}

// The gradient's workspace: partial gradients of B and C, then of A, D and dt_bias.
struct Partials {
  size_t bc, a, d;      // floats of one of each
  Partials(const ScanArgs& p, int blocks) : bc((size_t)blocks * p.batch * p.L * p.G * p.N), a((size_t)p.batch * p.channels * p.N), d((size_t)p.batch * p.channels) {}
  size_t bytes() const { return sizeof(float) * (2 * bc + a + 2 * d); }
};

// The rest of the gradient, in one launch.  blockIdx.y 0 and 1: a group's partial gradients of B and C, one from each of its workgroups, added up; 0 behind the end of a sequence.  2: those of
// A, D and dt_bias, one from each sequence.
template <typename T>
__global__ __launch_bounds__(256) void scan_join_kernel(ScanArgs p, T* gB, T* gC, float* gA, float* gD, float* gbias) {
  constexpr int U = 8;
  const long i = blockIdx.x * 256L + threadIdx.x;
  const float* part;
  long count, apart;      // terms, and how far they lie from each other
  if (blockIdx.y == 2) {
    const long states = (long)p.channels * p.N, at = i - states;
    apart = at < 0 ? states : p.channels, count = p.batch;
    part = at < 0 ? p.a_part + i : at < p.channels ? p.d_part + at : p.bias_part + (at - p.channels);
    float* out = at < 0 ? gA : at < p.channels ? gD : gbias;
    if (at >= 2L * p.channels || !out) return;
  } else {
    const long row = (long)p.G * p.N;
    apart = (long)p.batch * p.L * row;
    if (i >= apart || !(blockIdx.y ? gC : gB)) return;
    const long bt = i / row;
    const int b = bt / p.L, t = bt - (long)b * p.L;
    count = t < scan_length(p, b) ? p.blocks : 0;
    part = (blockIdx.y ? p.c_part : p.b_part) + i;
  }
  // eight sums, joined in a tree: one sum of thousands of channels in a row was off by 1.3e-6 of itself
  float sums[U];
#pragma unroll
  for (int u = 0; u < U; ++u) sums[u] = 0.f;
  for (long k = 0; k < count; k += U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = part[min(k + u, count - 1) * apart];
#pragma unroll
    for (int u = 0; u < U; ++u) sums[u] += k + u < count ? v[u] : 0.f;
  }
  const float sum = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
  if (blockIdx.y == 2) {
    const long states = (long)p.channels * p.N, at = i - states;
    if (at < 0) gA[i] = sum;
    else if (at < p.channels) gD[at] = sum;
    else gbias[at - p.channels] = sum;
  } else {
    (blockIdx.y ? gC : gB)[i] = value_to<T>(sum);
  }
}

}  // namespace
}  // namespace m2

using namespace m2;

// Positions between the states that are kept for the gradient.
extern "C" int m2_selective_scan_span(int N) {
  if (N < 1 || N > kMaxStates) return 0;
  return N <= 64 ? 64 : 32;
}

namespace {

void fill(ScanArgs& p, const m2_scan_inputs* in) {
  p.x = in->x, p.dt = in->dt, p.z = in->z, p.Bm = in->Bm, p.Cm = in->Cm;
  p.x_batch = in->x_batch, p.x_row = in->x_row, p.dt_batch = in->dt_batch, p.dt_row = in->dt_row, p.z_batch = in->z_batch, p.z_row = in->z_row;
  p.b_batch = in->b_batch, p.b_row = in->b_row, p.b_group = in->b_group, p.c_batch = in->c_batch, p.c_row = in->c_row, p.c_group = in->c_group;
  p.A = in->A, p.D = in->D, p.dt_bias = in->dt_bias, p.state = in->state, p.lengths = in->lengths;
  p.batch = in->batch, p.L = in->length, p.channels = in->channels, p.G = in->groups, p.N = in->states, p.softplus = in->softplus;
  p.per_group = p.G > 0 ? p.channels / p.G : 0;
}
bool given(const ScanArgs& p) { return p.x && p.dt && p.Bm && p.Cm && p.A; }

}  // namespace

extern "C" int m2_selective_scan_plan(int batch, int length, int channels, int groups, int states, int backward, int* plan) {
  if (!plan) return set_error(M2_ERR_ARG, "selective_scan_plan: null pointer");
  ScanArgs p{};
  p.batch = batch, p.L = length, p.channels = channels, p.G = groups, p.N = states;
  if (int rc = check_scan("selective_scan_plan", p, M2_DTYPE_F32)) return rc;
  const ScanPlan r = (backward ? bwd_plan : fwd_plan)(batch, length, channels, groups, states);
  if (int rc = check_grid("selective_scan_plan", p, r)) return rc;
  plan[0] = r.NS, plan[1] = r.NL, plan[2] = r.W, plan[3] = r.blocks * groups * batch, plan[4] = backward ? r.sets : 1;
  return M2_OK;
}

extern "C" int m2_selective_scan_fwd(const m2_scan_inputs* in, void* y, float* state_out, float* saved, int dtype, void* stream) {
  ScanArgs p{};
  if (in) fill(p, in);
  if (!in || !y || !given(p)) return set_error(M2_ERR_ARG, "selective_scan_fwd: null pointer");
  if (int rc = check_scan("selective_scan_fwd", p, dtype)) return rc;
  const ScanPlan plan = fwd_plan(p.batch, p.L, p.channels, p.G, p.N);
  p.y = y, p.state_out = state_out, p.saved = saved, p.blocks = plan.blocks;
  p.apart = m2_selective_scan_span(p.N), p.parts = (p.L + p.apart - 1) / p.apart;
  if (int rc = check_grid("selective_scan_fwd", p, plan)) return rc;
  const unsigned grid = (unsigned)((long)plan.blocks * p.G * p.batch);
  const size_t lds = fwd_lds(plan);
  int rc = M2_OK;
  with_scan_shape<ForwardShapes>(plan.NS, plan.NL, [&](auto ns, auto nl) {
    const auto launch = [&](auto t) {
      const auto kernel = selective_scan_kernel<decltype(t), decltype(ns)::value, decltype(nl)::value>;
      const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) {
        rc = set_error(M2_ERR_LAUNCH, "selective_scan_fwd: %zu bytes of shared memory: %s", lds, hipGetErrorString(e));
        return;
      }
      hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * plan.W), lds, (hipStream_t)stream, p);
    };
    if (dtype == M2_DTYPE_F32) launch(float{});
    else launch(uint16_t{});
  });
  return rc != M2_OK ? rc : check_launch("selective_scan_kernel");
}

extern "C" size_t m2_selective_scan_bwd_workspace_bytes(int batch, int length, int channels, int groups, int states) {
  ScanArgs p{};
  p.batch = batch, p.L = length, p.channels = channels, p.G = groups, p.N = states;
  if (check_scan("selective_scan_bwd", p, M2_DTYPE_F32)) return 0;
  return Partials(p, bwd_plan(batch, length, channels, groups, states).blocks).bytes();
}

extern "C" int m2_selective_scan_bwd(const m2_scan_inputs* in, const m2_scan_gradients* out, const float* saved, void* workspace, int dtype, void* stream) {
  ScanArgs p{};
  if (in) fill(p, in);
  if (!in || !out || !given(p) || !out->gy || !saved || !workspace) return set_error(M2_ERR_ARG, "selective_scan_bwd: null pointer");
  if (int rc = check_scan("selective_scan_bwd", p, dtype)) return rc;
  const ScanPlan plan = bwd_plan(p.batch, p.L, p.channels, p.G, p.N);
  if (int rc = check_grid("selective_scan_bwd", p, plan)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  p.blocks = plan.blocks, p.sets = plan.sets, p.apart = m2_selective_scan_span(p.N), p.parts = (p.L + p.apart - 1) / p.apart;
  p.gy = out->gy, p.gy_batch = out->gy_batch, p.gy_row = out->gy_row, p.gstate_out = out->gstate_out;
  p.gx = out->gx, p.gdt = out->gdt, p.gz = out->gz, p.gstate = out->gstate;
  p.saved = const_cast<float*>(saved);
  const Partials room(p, plan.blocks);
  p.b_part = static_cast<float*>(workspace), p.c_part = p.b_part + room.bc;
  p.a_part = p.c_part + room.bc, p.d_part = p.a_part + room.a, p.bias_part = p.d_part + room.d;
  if (int rc = scan_bwd(p, plan, dtype, s)) return rc;
  const long count = std::max((long)p.batch * p.L * p.G * p.N, (long)p.channels * (p.N + 2));
  const dim3 grid((unsigned)((count + 255) / 256), 3);
  if (dtype == M2_DTYPE_F32) hipLaunchKernelGGL(scan_join_kernel<float>, grid, dim3(256), 0, s, p, (float*)out->gB, (float*)out->gC, out->gA, out->gD, out->gdt_bias);
  else hipLaunchKernelGGL(scan_join_kernel<uint16_t>, grid, dim3(256), 0, s, p, (uint16_t*)out->gB, (uint16_t*)out->gC, out->gA, out->gD, out->gdt_bias);
  return check_launch("scan_join_kernel");
}

extern "C" int m2_selective_scan_step(const m2_scan_inputs* in, void* y, float* state_out, int dtype, void* stream) {
  ScanArgs p{};
  if (in) fill(p, in);
  if (!in || !y || !state_out || !given(p) || !p.state) return set_error(M2_ERR_ARG, "selective_scan_step: null pointer");
  if (int rc = check_scan("selective_scan_step", p, dtype)) return rc;
  p.y = y, p.state_out = state_out;
  const bool wide = p.N % 4 == 0 && m2::aligned16(p.A, p.state, p.state_out);
  const int P = std::min(64, pow2_from(wide ? p.N / 4 : p.N));
  const long groups = ((long)p.batch * p.channels * P + 255) / 256;
  if (groups >= 1L << 24) return set_error(M2_ERR_ARG, "selective_scan_step: B=%d, D=%d, N=%d are more than a launch holds", p.batch, p.channels, p.N);
  // 64 x 3584 x 64: 35.3 us with one channel a thread, 33.1 (3.6 TB/s) with two, 41 with four
  const int I = groups >= 16L * num_cus() ? 2 : 1;
  const auto launch = [&](auto t) {
    using T = decltype(t);
    const dim3 grid((unsigned)((groups + I - 1) / I));
    if (wide && I == 2) hipLaunchKernelGGL((selective_scan_step_kernel<T, 4, 2>), grid, dim3(256), 0, (hipStream_t)stream, p, P);
    else if (wide) hipLaunchKernelGGL((selective_scan_step_kernel<T, 4, 1>), grid, dim3(256), 0, (hipStream_t)stream, p, P);
    else if (I == 2) hipLaunchKernelGGL((selective_scan_step_kernel<T, 1, 2>), grid, dim3(256), 0, (hipStream_t)stream, p, P);
    else hipLaunchKernelGGL((selective_scan_step_kernel<T, 1, 1>), grid, dim3(256), 0, (hipStream_t)stream, p, P);
    return check_launch("selective_scan_step_kernel");
  };
  return dtype == M2_DTYPE_F32 ? launch(float{}) : launch(uint16_t{});
}
