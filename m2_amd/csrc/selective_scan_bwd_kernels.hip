// The gradient of the selective state space scan (selective_scan_kernels.hip).
//
//   u[t] = gy[t] silu(z[t])     dh[t, n] = C[t, n] u[t] + a[t + 1, n] dh[t + 1, n], with the gradient of the last state behind the last     a = exp(d A)
//   gB[t, n] = sum over channels dh d x     gC[t, n] = sum over channels u h     gx = d sum_n dh B + D u
//   gd = sum_n dh a h[t - 1] A + x sum_n dh B     gA = sum_t dh a h[t - 1] d     gD = sum_t u x     gz = gy (sum_n C h + D x) silu'(z)
//
// A workgroup goes through a sequence from its end, a step of 16 positions a wave at a time, each from the state that the forward has kept ahead of it, and in a step
// through several sets of 64 / NS channels.  A wave forms decays and inputs of its positions, runs over them from zero in both directions, and meets the others once,
// in shared memory, for the state it starts with and the gradient it ends with.  Forward again for the states, then backward: what the channels of a wave add to
// B's and C's gradients is summed across lanes as it arises, in a tree over positions that leaves each lane with positions of its own, and over the sets in shared
// memory; the sums of a workgroup go to memory for scan_join_kernel.  All in a fixed order.
//
// Bound by vector instructions (82 % of the cycles): 17 for each state and position, 9 in the trees' sums across lanes, 5 for each lane's own positions.  8 x 2048 x 1536, bf16, 16 states: 462 us of the
// 668 that forward and gradient take, 404 MB in 79.  Partial gradients of B and C are 2 x 100 MB (two sets a workgroup; 34 us to join them).  Registers: loads of four positions' shared values at a time, and
// arguments read anew where they are used (236 -> 162, three waves a SIMD; 436 moves of spilled scalars gone).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "selective_scan.h"

namespace m2 {

// Values of the positions of a group of 2^LV, highest first, summed across 2^LV lanes: position bit k goes with lane bit FIRST + k * STEP, and each lane is left with the
// sum of its own position.
template <int LV, int NL, int FIRST, int STEP>
struct Tree {
  float at[LV > 0 ? LV : 1][NL];      // per level, what waits for its neighbour
  // position T of the group; v is complete when T is 0
  template <int T, int K = 0>
  __device__ __forceinline__ void add(float (&v)[NL], int lane) {
    if constexpr (K < LV) {
      if constexpr ((T >> K) & 1) {
#pragma unroll
        for (int j = 0; j < NL; ++j) at[K][j] = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < NL; ++j) v[j] = split_over_bit<FIRST + K * STEP>(v[j], at[K][j], lane);
        add<T, K + 1>(v, lane);
      }
    }
  }
};
// Keeps the loads of a group of positions behind those before it: all of them ahead of their use would not fit into registers.
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }

template <int FIRST, int LAST, typename F>
__device__ __forceinline__ void count_down(F&& f) {      // f(FIRST), ..., f(LAST) as constants
  f(std::integral_constant<int, FIRST>{});
  if constexpr (FIRST > LAST) count_down<FIRST - 1, LAST>(f);
}

// Floats of shared memory: of a wave, of a wave and set, of a set.
template <int NS, int NL>
struct GradientRoom {
  using S = ScanShape<NS, NL>;
  static constexpr int kChannels = S::CW * S::PITCH;
  static constexpr int kWave = 4 * S::TILE + 3 * kChannels + 2 * 3 * 64 * NL;      // B, C and their gradients, d, d x, u, and the turns of what passes between waves
  static constexpr int kWaveSet = 64 * (NL + 2);                                   // gradients of A, D, dt_bias
  static constexpr int kSet = 2 * 64 * NL;                                         // what reaches the step behind, in two turns
};

// (read, added and written: an atomic addition in shared memory takes 200 cycles a wave)
template <int NL>
__device__ __forceinline__ void add_shared(float* p, const float (&v)[NL]) {
  float sum[NL];
  load_values<float, NL>(p, sum);
#pragma unroll
  for (int j = 0; j < NL; ++j) sum[j] += v[j];
  store_values<float, NL>(p, sum);
}

template <typename T, int NS, int NL>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(NL == 2 && NS > 4 && (NS != 32 || sizeof(T) == 2) ? 3 : 2))) void selective_scan_bwd_kernel(ScanArgs p) {
  static_assert(NS >= 2, "the sums over channels take up to five lane bits");
  using S = ScanShape<NS, NL>;
  using Room = GradientRoom<NS, NL>;
  constexpr int CW = S::CW, NP = S::NP, TT = S::TT, NT = S::NT, PITCH = S::PITCH;
  constexpr int CBITS = log2_of(CW), LV = CBITS < 4 ? CBITS : 4;      // lane bits of channels; those that go with positions
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane / NS, q = lane % NS;
  const int id = xcd_order(blockIdx.x, gridDim.x), block = id % p.blocks, g = id / p.blocks % p.G, b = id / p.blocks / p.G;
  const int n = scan_length(p, b), span = W * TT;
  const int sets = min(p.sets, (p.per_group - block * p.sets * CW + CW - 1) / CW);
  float* Bs = lds + w * Room::kWave;
  float* Cs = Bs + S::TILE;
  float* gBs = Cs + S::TILE;
  float* gCs = gBs + S::TILE;
  float* ds = gCs + S::TILE;
  float* xs = ds + Room::kChannels;
  float* us = xs + Room::kChannels;
  float* ex = lds + W * (Room::kWave - 2 * 3 * 64 * NL);      // (2, W, 3, 64, NL), behind the waves' own
  float* mine = lds + W * Room::kWave + w * p.sets * Room::kWaveSet;
  float* carried = lds + W * (Room::kWave + p.sets * Room::kWaveSet);
  // (the waves' own tiles lie one behind the other without the turns)
  {
    const int shift = w * 2 * 3 * 64 * NL;
    Bs -= shift, Cs -= shift, gBs -= shift, gCs -= shift, ds -= shift, xs -= shift, us -= shift;
  }
  const bool moves = NS <= TT || q < TT;
  const int q0 = NS <= TT ? q : min(q, TT - 1);
  const auto channel = [&](int set, bool& on) {
    const ArgsInMemory& p = *arguments_anew();
    const int first = (block * p.sets + set) * CW, count = min(CW, p.per_group - first);
    on = c < count;
    return g * p.per_group + first + min(c, count - 1);
  };

  for (int i = lane; i < 2 * S::TILE; i += 64) gBs[i] = 0.f;
  for (int i = lane; i < sets * Room::kWaveSet; i += 64) mine[i] = 0.f;
  if (w == 0)
    for (int set = 0; set < sets; ++set) {
      bool on;
      const int ch = channel(set, on);
#pragma unroll
      for (int j = 0; j < NL; ++j)
#pragma unroll
        for (int turn = 0; turn < 2; ++turn)
          carried[((set * 2 + turn) * 64 + lane) * NL + j] = on && q * NL + j < p.N && p.gstate_out ? p.gstate_out[((long)b * p.channels + ch) * p.N + q * NL + j] : 0.f;
    }

  const int steps = (n + span - 1) / span;
  const bool gated = p.z, soft = p.softplus, biased = p.dt_bias, skips = p.D;
  const int N = p.N;

  T rx[NT], rdt[NT], rz[NT], rg[NT];
  float rA[NL], rH[NL], rbias, rskip;
  TileIn<T, NS, NL, S::AHEAD ? S::NB : 1> rb, rc;
  const auto load = [&](int s, int set) {
    ArgsInMemory& p = *arguments_anew();
    bool on;
    const int ch = channel(set, on), t0 = min(s * span + w * TT, n - 1), last = min(n - 1 - t0, TT - 1);
    const auto rows = [&](T (&r)[NT], const void* tensor, long batch, long row) {
      const T* base = static_cast<const T*>(tensor) + b * batch + t0 * row;
      const Near off = Near::of(base, q0, row, ch, last);
#pragma unroll
      for (int i = 0; i < NT; ++i) r[i] = at_offset<const T>(base, off((uint32_t)(i * NS * sizeof(T)) * (uint32_t)row));
    };
    rows(rx, p.x, p.x_batch, p.x_row);
    rows(rdt, p.dt, p.dt_batch, p.dt_row);
    rows(rg, p.gy, p.gy_batch, p.gy_row);
    rows(rz, p.z ? p.z : p.x, p.z ? p.z_batch : p.x_batch, p.z ? p.z_row : p.x_row);      // (no gate: loads that nothing comes of, rather than waits around a branch)
    const float* kept = p.saved + ((long)b * p.parts + s) * p.channels * p.N;
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const uint32_t at = (__umul24((uint32_t)ch, (uint32_t)p.N) + (uint32_t)min(q * NL + j, p.N - 1)) * 4u;
      rA[j] = at_offset<const float>(p.A, at), rH[j] = at_offset<const float>(kept, at);
    }
    // (without a bias or D: a value that is not used)
    rbias = at_offset<const float>(p.dt_bias ? p.dt_bias : p.A, (uint32_t)ch * 4u);
    rskip = at_offset<const float>(p.D ? p.D : p.A, (uint32_t)ch * 4u);
  };
  const auto load_tiles = [&](int s) {
    ArgsInMemory& p = *arguments_anew();
    const int t0 = min(s * span + w * TT, n - 1);
    rb.load(static_cast<const T*>(p.Bm) + b * p.b_batch + g * p.b_group, p.b_row, t0, n, p.N, lane);
    rc.load(static_cast<const T*>(p.Cm) + b * p.c_batch + g * p.c_group, p.c_row, t0, n, p.N, lane);
  };
  if (steps > 0) {
    load(steps - 1, 0);
    if constexpr (S::AHEAD) load_tiles(steps - 1);
  }
  __syncthreads();
  int turn = 0;
  for (int s = steps - 1; s >= 0; --s) {
    const int t0 = s * span + w * TT;
    wave_sync();      // the tiles have been read
    if constexpr (S::AHEAD) {
      rb.put(Bs, N, lane);
      rc.put(Cs, N, lane);
      load_tiles(max(s - 1, 0));
    } else {
      ArgsInMemory& p = *arguments_anew();
      tile_in<T, NS, NL>(Bs, static_cast<const T*>(p.Bm) + b * p.b_batch + g * p.b_group, p.b_row, min(t0, n - 1), n, p.N, lane);
      tile_in<T, NS, NL>(Cs, static_cast<const T*>(p.Cm) + b * p.c_batch + g * p.c_group, p.c_row, min(t0, n - 1), n, p.N, lane);
    }
    for (int set = 0; set < sets; ++set, turn ^= 1) {
      bool on;
      const int ch = channel(set, on);
      float A[NL], start[NL], xv[NT], d[NT], d_slope[NT], gv[NT], u[NT], gz[NT], own_total = 0.f;
      float skip = skips ? rskip : 0.f;
      const float bias = biased ? rbias : 0.f;
      made_here(skip);
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const bool real = on && q * NL + j < N;
        A[j] = real ? rA[j] : 0.f, start[j] = real ? rH[j] : 0.f;
        made_here(A[j]), made_here(start[j]);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const bool inside = on && t0 + q0 + i * NS < n;
        const float raw = value_of<T>(rdt[i]) + bias;
        d[i] = raw, d_slope[i] = inside ? 1.f : 0.f;
        if (soft) {
          const Logistic<true> l(raw);
          d[i] = softplus_of(raw, l.u);
          d_slope[i] = inside ? l.value() : 0.f;
        }
        d[i] = inside ? d[i] : 0.f;
        xv[i] = inside ? value_of<T>(rx[i]) : 0.f;
        gv[i] = inside ? value_of<T>(rg[i]) : 0.f;
        u[i] = gv[i], gz[i] = 0.f;
        if (gated) {
          const float zv = inside ? value_of<T>(rz[i]) : 0.f;
          const Logistic<sizeof(T) == 4> l(zv);
          u[i] = gv[i] * (zv * l.value());
          gz[i] = gv[i] * silu_slope_of(zv, l);
        }
        made_here(xv[i]), made_here(d[i]), made_here(d_slope[i]), made_here(u[i]), made_here(gz[i]);
        own_total += moves ? d[i] : 0.f;
        if (moves) ds[c * PITCH + q0 + i * NS] = d[i], xs[c * PITCH + q0 + i * NS] = d[i] * xv[i], us[c * PITCH + q0 + i * NS] = u[i];
      }
      wave_sync();
      load(set + 1 < sets ? s : max(s - 1, 0), set + 1 < sets ? set + 1 : 0);      // (the very last for nothing)
      const float total = lane_sum<NS>(own_total, lane);
      float a[TT][NL], h[TT][NL], last[NL], left[NL], A2[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) last[j] = left[j] = 0.f, A2[j] = decay_rate(A[j]);
#pragma unroll
      for (int t4 = 0; t4 < TT; t4 += 4) {
        keep_order();
        float d4[4], x4[4];
        load_values<float, 4>(ds + c * PITCH + t4, d4);
        load_values<float, 4>(xs + c * PITCH + t4, x4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = t4 + i;
          float bn[NL];
          load_values<float, NL>(Bs + t * NP + q * NL, bn);
#pragma unroll
          for (int j = 0; j < NL; ++j) {
            a[t][j] = __builtin_amdgcn_exp2f(d4[i] * A2[j]);
            h[t][j] = x4[i] * bn[j];      // (for now what the position puts in)
            last[j] = fmaf(a[t][j], last[j], h[t][j]);
          }
        }
      }
#pragma unroll
      for (int t4 = TT - 4; t4 >= 0; t4 -= 4) {
        keep_order();
        float u4[4];
        load_values<float, 4>(us + c * PITCH + t4, u4);
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          float cn[NL];
          load_values<float, NL>(Cs + (t4 + i) * NP + q * NL, cn);
#pragma unroll
          for (int j = 0; j < NL; ++j) left[j] = fmaf(cn[j], u4[i], left[j]) * a[t4 + i][j];
        }
      }
      // what the waves before and behind do to a state and to its gradient
      float P[NL], right[NL], R[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) P[j] = __builtin_amdgcn_exp2f(total * A2[j]);
      float* now = ex + turn * W * 3 * 64 * NL;
      store_values<float, NL>(now + (w * 3 * 64 + lane) * NL, P);
      store_values<float, NL>(now + ((w * 3 + 1) * 64 + lane) * NL, last);
      store_values<float, NL>(now + ((w * 3 + 2) * 64 + lane) * NL, left);
      __syncthreads();      // (two turns: what is written next is read behind the next barrier)
      load_values<float, NL>(carried + ((set * 2 + (s & 1)) * 64 + lane) * NL, R);
      for (int o = 0; o < w; ++o) {
        float po[NL], ho[NL];
        load_values<float, NL>(now + (o * 3 * 64 + lane) * NL, po);
        load_values<float, NL>(now + ((o * 3 + 1) * 64 + lane) * NL, ho);
#pragma unroll
        for (int j = 0; j < NL; ++j) start[j] = fmaf(po[j], start[j], ho[j]);
      }
      const auto meet = [&](int o) {
        float po[NL], lo[NL];
        load_values<float, NL>(now + (o * 3 * 64 + lane) * NL, po);
        load_values<float, NL>(now + ((o * 3 + 2) * 64 + lane) * NL, lo);
#pragma unroll
        for (int j = 0; j < NL; ++j) R[j] = fmaf(po[j], R[j], lo[j]);
      };
      for (int o = W - 1; o > w; --o) meet(o);
#pragma unroll
      for (int j = 0; j < NL; ++j) right[j] = R[j];
      if (w == 0) {      // the first wave has met all others
        meet(0);
        store_values<float, NL>(carried + ((set * 2 + (~s & 1)) * 64 + lane) * NL, R);
      }
      // the states
      {
        float run[NL];
#pragma unroll
        for (int j = 0; j < NL; ++j) run[j] = start[j];
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
          for (int j = 0; j < NL; ++j) h[t][j] = run[j] = fmaf(a[t][j], run[j], h[t][j]);
      }
      // sum_n dh B, sum_n dh a h A, sum_n C h of the lane's positions
      constexpr int QV = log2_of(NS) < 4 ? log2_of(NS) : 4;
      float into[NT], kept[NT], out[NT], gA[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) gA[j] = 0.f;
      Tree<LV, NL, 5, -1> tb, tc;
      Tree<QV, 3, 0, 1> tq;
      float d4[4], x4[4], u4[4];
      count_down<TT - 1, 0>([&](auto tt) {
        constexpr int t = decltype(tt)::value;
        if constexpr (t % 4 == 3) {
          keep_order();
          load_values<float, 4>(ds + c * PITCH + t - 3, d4);
          load_values<float, 4>(xs + c * PITCH + t - 3, x4);
          load_values<float, 4>(us + c * PITCH + t - 3, u4);
        }
        float bn[NL], cn[NL], vb[NL], vc[NL], vq[3];
        load_values<float, NL>(Bs + t * NP + q * NL, bn);
        load_values<float, NL>(Cs + t * NP + q * NL, cn);
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const float dh = fmaf(cn[j], u4[t % 4], right[j]);
          vb[j] = dh * x4[t % 4];
          vc[j] = u4[t % 4] * h[t][j];
          right[j] = dh * a[t][j];
          const float k = right[j] * (t > 0 ? h[t > 0 ? t - 1 : 0][j] : start[j]);
          vq[0] = j == 0 ? dh * bn[j] : fmaf(dh, bn[j], vq[0]);
          vq[1] = j == 0 ? k * A[j] : fmaf(k, A[j], vq[1]);
          vq[2] = j == 0 ? cn[j] * h[t][j] : fmaf(cn[j], h[t][j], vq[2]);
          gA[j] = fmaf(d4[t % 4], k, gA[j]);
        }
        tq.template add<t % (1 << QV)>(vq, lane);
        if constexpr (t % (1 << QV) == 0) {
          if constexpr (NS > 16) {      // (lanes beyond the positions)
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              vq[k] = sum_over_bit<4>(vq[k], lane);
              if constexpr (NS > 32) vq[k] = sum_over_bit<5>(vq[k], lane);
            }
          }
          into[t >> QV] = vq[0], kept[t >> QV] = vq[1], out[t >> QV] = vq[2];
        }
        tb.template add<t % (1 << LV)>(vb, lane);
        tc.template add<t % (1 << LV)>(vc, lane);
        if constexpr (t % (1 << LV) == 0) {
          // (two lanes a channel: the fifth bit of the channels)
          if constexpr (CBITS > 4) {
#pragma unroll
            for (int j = 0; j < NL; ++j) vb[j] = sum_over_bit<1>(vb[j], lane), vc[j] = sum_over_bit<1>(vc[j], lane);
          }
          int at = t;
#pragma unroll
          for (int k = 0; k < LV; ++k) at += ((lane >> (5 - k)) & 1) << k;
          if (CBITS <= 4 || (lane & 3) < NS) add_shared<NL>(gBs + at * NP + q * NL, vb), add_shared<NL>(gCs + at * NP + q * NL, vc);
        }
      });
      float gD = 0.f, gbias = 0.f;
      ArgsInMemory& p = *arguments_anew();
      const long out_at = ((long)b * p.L + t0) * p.channels;
      T* gx = static_cast<T*>(p.gx) + out_at;
      T* gdt = static_cast<T*>(p.gdt) + out_at;
      T* gzs = static_cast<T*>(p.gz) + out_at;
      const uint32_t off = (__umul24((uint32_t)q0, (uint32_t)p.channels) + (uint32_t)ch) * sizeof(T);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int t = t0 + i * NS;
        const bool inside = t + q0 < n;
        // (behind the end `kept` is what A makes of a state that stays, which may pass fp32's range)
        const float gxv = fmaf(d[i], into[i], skip * u[i]), gd = inside ? fmaf(xv[i], into[i], kept[i]) * d_slope[i] : 0.f;
        gD = fmaf(u[i], xv[i], gD);
        gbias += gd;
        if (on && moves && t + q0 < p.L) {
          const uint32_t at = off + (uint32_t)(i * NS * sizeof(T)) * (uint32_t)p.channels;
          if (p.gx) at_offset<T>(gx, at) = value_to<T>(inside ? gxv : 0.f);
          if (p.gdt) at_offset<T>(gdt, at) = value_to<T>(gd);
          if (p.gz) at_offset<T>(gzs, at) = value_to<T>(inside ? gz[i] * fmaf(skip, xv[i], out[i]) : 0.f);
        }
      }
      float* sums = mine + set * Room::kWaveSet + lane;
#pragma unroll
      for (int j = 0; j < NL; ++j) sums[j * 64] += gA[j];
      sums[NL * 64] += moves ? gD : 0.f;
      sums[(NL + 1) * 64] += moves ? gbias : 0.f;
      wave_sync();      // positions' values have been read
    }
    // the workgroup's part of B's and C's gradients
    ArgsInMemory& p = *arguments_anew();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float* sums = which ? gCs : gBs;
      float* out = (which ? p.c_part : p.b_part) + ((((long)block * p.batch + b) * p.L + t0) * p.G + g) * p.N;
      for (int i = lane; i < S::TILE; i += 64) {
        const int t = i / NP, at = i % NP;
        if (t0 + t < n && at < p.N) out[(long)t * p.G * p.N + at] = sums[i];
        sums[i] = 0.f;
      }
    }
  }
  const ArgsInMemory& end = *arguments_anew();
  for (int set = 0; set < sets; ++set) {
    bool on;
    const int ch = channel(set, on);
    for (int t0 = steps * span + w * TT; t0 < end.L; t0 += span)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int t = t0 + q0 + i * NS;
        const long at = ((long)b * end.L + t) * end.channels + ch;
        if (on && moves && t < end.L) {
          if (end.gx) static_cast<T*>(end.gx)[at] = value_to<T>(0.f);
          if (end.gdt) static_cast<T*>(end.gdt)[at] = value_to<T>(0.f);
          if (end.gz) static_cast<T*>(end.gz)[at] = value_to<T>(0.f);
        }
      }
  }
  // over the waves, and over a channel's lanes
  __syncthreads();
  for (int set = w; set < sets; set += W) {
    bool on;
    const int ch = channel(set, on);
    float sums[NL + 2];
#pragma unroll
    for (int j = 0; j < NL + 2; ++j) {
      sums[j] = 0.f;
      for (int o = 0; o < W; ++o) sums[j] += lds[W * Room::kWave + (o * end.sets + set) * Room::kWaveSet + j * 64 + lane];
    }
    const float gD = lane_sum<NS>(sums[NL], lane), gbias = lane_sum<NS>(sums[NL + 1], lane);
    if (!on) continue;
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const long at = ((long)b * end.channels + ch) * end.N + q * NL + j;
      if (q * NL + j >= end.N) continue;
      end.a_part[at] = sums[j];
      if (end.gstate) end.gstate[at] = carried[((set * 2 + 1) * 64 + lane) * NL + j];      // (behind step 0)
    }
    if (q == 0) end.d_part[(long)b * end.channels + ch] = gD, end.bias_part[(long)b * end.channels + ch] = gbias;
  }
}

size_t scan_bwd_lds(const ScanPlan& plan) {
  size_t bytes = 0;
  with_scan_shape<GradientShapes>(plan.NS, plan.NL, [&](auto ns, auto nl) {
    using Room = GradientRoom<decltype(ns)::value, decltype(nl)::value>;
    bytes = sizeof(float) * (plan.W * (Room::kWave + plan.sets * Room::kWaveSet) + plan.sets * Room::kSet);
  });
  return bytes;
}

int scan_bwd(const ScanArgs& p, const ScanPlan& plan, int dtype, hipStream_t stream) {
  const unsigned grid = (unsigned)((long)plan.blocks * p.G * p.batch);
  const size_t lds = scan_bwd_lds(plan);
  int rc = M2_OK;
  with_scan_shape<GradientShapes>(plan.NS, plan.NL, [&](auto ns, auto nl) {
    const auto launch = [&](auto t) {
      const auto kernel = selective_scan_bwd_kernel<decltype(t), decltype(ns)::value, decltype(nl)::value>;
      const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) {
        rc = set_error(M2_ERR_LAUNCH, "selective_scan_bwd: %zu bytes of shared memory: %s", lds, hipGetErrorString(e));
        return;
      }
      hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * plan.W), lds, stream, p);
    };
    if (dtype == M2_DTYPE_F32) launch(float{});
    else launch(uint16_t{});
  });
  return rc != M2_OK ? rc : check_launch("selective_scan_bwd_kernel");
}

}  // namespace m2
