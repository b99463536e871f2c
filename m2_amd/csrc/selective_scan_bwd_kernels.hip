// The gradient of the selective state space scan (selective_scan_kernels.hip).
//
//   u[t] = gy[t] silu(z[t])     dh[t, n] = C[t, n] u[t] + a[t + 1, n] dh[t + 1, n], with the gradient of the last state behind the last     a = exp(d A)
//   gB[t, n] = sum over channels dh d x     gC[t, n] = sum over channels u h     gx = d sum_n dh B + D u
//   gd = sum_n dh a h[t - 1] A + x sum_n dh B     gA = sum_t dh a h[t - 1] d     gD = sum_t u x     gz = gy (sum_n C h + D x) silu'(z)
//
// Workgroups lie as in the forward and go through a sequence from its end, a step of `span` positions at a time, each from the state that the forward has kept ahead
// of it.  A wave forms decays and inputs of its positions, runs over them from zero in both directions, and meets the others once, in shared memory, for the state it
// starts with and the gradient it ends with.  Forward again for the states, then backward: what the channels of a wave add to B's and C's gradients is summed
// across lanes as it arises, in a tree over positions that leaves each lane with positions of its own, and goes to memory for scan_join_kernel, in a fixed order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "selective_scan.h"

namespace m2 {

// Values of the positions of a group of 2^LV, highest first, summed across the lanes of the wave's channels: position bit k goes with lane bit 5 - k.
template <int LV, int NL>
struct Tree {
  float at[LV > 0 ? LV : 1][NL];      // per level, what waits for its neighbour
  // position t of the group; the result is complete in v when t is 0
  template <int T>
  __device__ __forceinline__ void add(float (&v)[NL], int lane) {
    step<T, 0>(v, lane);
  }
  template <int T, int K>
  __device__ __forceinline__ void step(float (&v)[NL], int lane) {
    if constexpr (K < LV) {
      if constexpr ((T >> K) & 1) {
#pragma unroll
        for (int j = 0; j < NL; ++j) at[K][j] = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < NL; ++j) v[j] = split_over_bit<5 - K>(v[j], at[K][j], lane);
        step<T, K + 1>(v, lane);
      }
    }
  }
};

template <int FIRST, int LAST, typename F>
__device__ __forceinline__ void count_down(F&& f) {      // f(FIRST), ..., f(LAST) as constants
  f(std::integral_constant<int, FIRST>{});
  if constexpr (FIRST > LAST) count_down<FIRST - 1, LAST>(f);
}

template <typename T, int NS, int NL>
__global__ __launch_bounds__(512) void selective_scan_bwd_kernel(ScanArgs p) {
  static_assert(NS >= 2, "the sums over channels take up to five lane bits");
  using S = ScanShape<NS, NL>;
  constexpr int CW = S::CW, NP = S::NP, TT = S::TT, NT = S::NT, PITCH = S::PITCH;
  constexpr int CBITS = log2_of(CW), LV = CBITS < 4 ? CBITS : 4;      // lane bits of channels; those that go with positions
  constexpr int kWave = 2 * S::TILE + 3 * CW * PITCH;
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane / NS, q = lane % NS;
  const int id = xcd_order(blockIdx.x, gridDim.x), block = id % p.blocks, g = id / p.blocks % p.G, b = id / p.blocks / p.G;
  const int count = min(CW, p.per_group - block * CW);
  const bool on = c < count;
  const int ch = g * p.per_group + block * CW + min(c, count - 1);
  const int n = scan_length(p, b), span = W * TT;
  float* Bs = lds + w * kWave;
  float* Cs = Bs + S::TILE;
  float* ds = Cs + S::TILE;
  float* xs = ds + CW * PITCH;
  float* us = xs + CW * PITCH;
  float* ex = lds + W * kWave;      // (2, W, 3, 64, NL)

  float A[NL], R[NL], gA[NL];      // R: the gradient of the state behind the step, times the decay there
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int at = q * NL + j;
    const bool real = on && at < p.N;
    A[j] = real ? p.A[(long)ch * p.N + at] : 0.f;
    R[j] = real && p.gstate_out ? p.gstate_out[((long)b * p.channels + ch) * p.N + at] : 0.f;
    gA[j] = 0.f;
  }
  const float bias = p.dt_bias ? p.dt_bias[ch] : 0.f, skip = p.D ? p.D[ch] : 0.f;
  const T* x = static_cast<const T*>(p.x) + b * p.x_batch + ch;
  const T* dt = static_cast<const T*>(p.dt) + b * p.dt_batch + ch;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_batch + ch : nullptr;
  const T* gy = static_cast<const T*>(p.gy) + b * p.gy_batch + ch;
  const T* Bm = static_cast<const T*>(p.Bm) + b * p.b_batch + g * p.b_group;
  const T* Cm = static_cast<const T*>(p.Cm) + b * p.c_batch + g * p.c_group;
  const long out_at = (long)b * p.L * p.channels + ch;
  const bool moves = NS <= TT || q < TT;
  const int q0 = NS <= TT ? q : min(q, TT - 1);
  const long bc_at = (((long)block * p.batch + b) * p.L * p.G + g) * p.N, bc_row = (long)p.G * p.N;      // of partial gradients of B and C

  T rx[NT], rdt[NT], rz[NT], rg[NT];
  const auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int t = min(t0 + q0 + i * NS, n - 1);
      rx[i] = x[t * p.x_row], rdt[i] = dt[t * p.dt_row], rg[i] = gy[t * p.gy_row];
      if (z) rz[i] = z[t * p.z_row];
    }
  };
  const int steps = (n + span - 1) / span;
  if (steps > 0) load((steps - 1) * span + w * TT);
  float gD = 0.f, gbias = 0.f;
  for (int s = steps - 1; s >= 0; --s) {
    const int t0 = s * span + w * TT;
    float H[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int at = q * NL + j;
      H[j] = on && at < p.N ? p.saved[(((long)b * p.parts + s) * p.channels + ch) * p.N + at] : 0.f;
    }
    float xv[NT], raw[NT], own_d[NT], zv[NT], gv[NT], u[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const bool inside = on && t0 + q0 + i * NS < n;
      raw[i] = value_of<T>(rdt[i]) + bias;
      own_d[i] = inside ? (p.softplus ? softplus(raw[i]) : raw[i]) : 0.f;
      xv[i] = inside ? value_of<T>(rx[i]) : 0.f;
      gv[i] = inside ? value_of<T>(rg[i]) : 0.f;
      zv[i] = z && inside ? value_of<T>(rz[i]) : 0.f;
      u[i] = z ? gv[i] * silu(zv[i]) : gv[i];
    }
    wave_sync();      // the tiles have been read
    tile_in<T, NS, NL>(Bs, Bm, p.b_row, t0, n, p.N, lane);
    tile_in<T, NS, NL>(Cs, Cm, p.c_row, t0, n, p.N, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (moves) ds[c * PITCH + q0 + i * NS] = own_d[i], xs[c * PITCH + q0 + i * NS] = own_d[i] * xv[i], us[c * PITCH + q0 + i * NS] = u[i];
    wave_sync();
    if (s > 0) load(t0 - span);
    float a[TT][NL], h[TT][NL], last[NL], left[NL], total = 0.f;
#pragma unroll
    for (int j = 0; j < NL; ++j) last[j] = left[j] = 0.f;
#pragma unroll
    for (int t4 = 0; t4 < TT; t4 += 4) {
      float d4[4], x4[4];
      load_values<float, 4>(ds + c * PITCH + t4, d4);
      load_values<float, 4>(xs + c * PITCH + t4, x4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t4 + i;
        float bn[NL];
        load_values<float, NL>(Bs + t * NP + q * NL, bn);
        total += d4[i];
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          a[t][j] = __builtin_amdgcn_exp2f(d4[i] * (A[j] * kLog2E));
          h[t][j] = x4[i] * bn[j];      // (for now what the position puts in)
          last[j] = fmaf(a[t][j], last[j], h[t][j]);
        }
      }
    }
#pragma unroll
    for (int t4 = TT - 4; t4 >= 0; t4 -= 4) {
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
    float P[NL], start[NL], right[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) P[j] = __builtin_amdgcn_exp2f(total * (A[j] * kLog2E)), start[j] = H[j], right[j] = R[j];
    float* turn = ex + (s & 1) * W * 3 * 64 * NL;
    store_values<float, NL>(turn + (w * 3 * 64 + lane) * NL, P);
    store_values<float, NL>(turn + ((w * 3 + 1) * 64 + lane) * NL, last);
    store_values<float, NL>(turn + ((w * 3 + 2) * 64 + lane) * NL, left);
    __syncthreads();      // (two turns: what is written next is read behind the next barrier)
    for (int o = 0; o < w; ++o) {
      float po[NL], ho[NL];
      load_values<float, NL>(turn + (o * 3 * 64 + lane) * NL, po);
      load_values<float, NL>(turn + ((o * 3 + 1) * 64 + lane) * NL, ho);
#pragma unroll
      for (int j = 0; j < NL; ++j) start[j] = fmaf(po[j], start[j], ho[j]);
    }
    for (int o = W - 1; o >= 0; --o) {
      if (o == w) {
#pragma unroll
        for (int j = 0; j < NL; ++j) right[j] = R[j];
      }
      float po[NL], lo[NL];
      load_values<float, NL>(turn + (o * 3 * 64 + lane) * NL, po);
      load_values<float, NL>(turn + ((o * 3 + 2) * 64 + lane) * NL, lo);
#pragma unroll
      for (int j = 0; j < NL; ++j) R[j] = fmaf(po[j], R[j], lo[j]);
    }
    // the states, and the outputs where a gate asks for them
    float out[TT];
    {
      float run[NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) run[j] = start[j];
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int j = 0; j < NL; ++j) h[t][j] = run[j] = fmaf(a[t][j], run[j], h[t][j]);
    }
    if (z) {
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float cn[NL];
        load_values<float, NL>(Cs + t * NP + q * NL, cn);
        out[t] = cn[0] * h[t][0];
#pragma unroll
        for (int j = 1; j < NL; ++j) out[t] = fmaf(cn[j], h[t][j], out[t]);
      }
      share_positions<NS, 0>(out, lane);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int t = t0 + q0 + i * NS;
        if (p.gz && on && moves && t < p.L) static_cast<T*>(p.gz)[out_at + (long)t * p.channels] = value_to<T>(gv[i] * fmaf(skip, xv[i], out[i]) * silu_slope(zv[i]));
      }
    }
    float into[TT];      // sum_n dh B; out: sum_n dh a h A
    Tree<LV, NL> tb, tc;
    count_down<TT - 1, 0>([&](auto tt) {
      constexpr int t = decltype(tt)::value;
      const float d = ds[c * PITCH + t], dx = xs[c * PITCH + t], ut = us[c * PITCH + t];
      float bn[NL], cn[NL], vb[NL], vc[NL];
      load_values<float, NL>(Bs + t * NP + q * NL, bn);
      load_values<float, NL>(Cs + t * NP + q * NL, cn);
      into[t] = out[t] = 0.f;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const float dh = fmaf(cn[j], ut, right[j]);
        vb[j] = dh * dx;
        vc[j] = ut * h[t][j];
        into[t] = fmaf(dh, bn[j], into[t]);
        right[j] = dh * a[t][j];
        const float k = right[j] * (t > 0 ? h[t > 0 ? t - 1 : 0][j] : start[j]);
        out[t] = fmaf(k, A[j], out[t]);
        gA[j] = fmaf(d, k, gA[j]);
      }
      tb.template add<t % (1 << LV)>(vb, lane);
      tc.template add<t % (1 << LV)>(vc, lane);
      if constexpr (t % (1 << LV) == 0) {
        // (two lanes a channel: the fifth bit of the channels)
        if constexpr (CBITS > 4) {
#pragma unroll
          for (int j = 0; j < NL; ++j) vb[j] = sum_over_bit<1>(vb[j], lane), vc[j] = sum_over_bit<1>(vc[j], lane);
        }
        int mine = t0 + t;
#pragma unroll
        for (int k = 0; k < LV; ++k) mine += ((lane >> (5 - k)) & 1) << k;
        if (mine < n && (CBITS <= 4 || (lane & 3) < NS)) {
          const long at = bc_at + mine * bc_row + q * NL;
#pragma unroll
          for (int j = 0; j < NL; ++j)
            if (q * NL + j < p.N) p.b_part[at + j] = vb[j], p.c_part[at + j] = vc[j];
        }
      }
    });
    share_positions<NS, 0>(into, lane);
    share_positions<NS, 0>(out, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int t = t0 + q0 + i * NS;
      const bool inside = t < n;
      const float gx = fmaf(own_d[i], into[i], skip * u[i]);
      float gd = fmaf(xv[i], into[i], out[i]);
      if (p.softplus) gd *= sigmoid(raw[i]);
      if (!inside) gd = 0.f;
      if (on && moves) {
        gD = fmaf(u[i], xv[i], gD);
        gbias += gd;
        if (t < p.L) {
          if (p.gx) static_cast<T*>(p.gx)[out_at + (long)t * p.channels] = value_to<T>(inside ? gx : 0.f);
          if (p.gdt) static_cast<T*>(p.gdt)[out_at + (long)t * p.channels] = value_to<T>(gd);
        }
      }
    }
  }
  for (int t0 = steps * span + w * TT; t0 < p.L; t0 += span)
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int t = t0 + q0 + i * NS;
      if (on && moves && t < p.L) {
        if (p.gx) static_cast<T*>(p.gx)[out_at + (long)t * p.channels] = value_to<T>(0.f);
        if (p.gdt) static_cast<T*>(p.gdt)[out_at + (long)t * p.channels] = value_to<T>(0.f);
        if (p.gz) static_cast<T*>(p.gz)[out_at + (long)t * p.channels] = value_to<T>(0.f);
      }
    }
  // over a channel's lanes, then over the waves
  gD = lane_sum<NS>(gD, lane);
  gbias = lane_sum<NS>(gbias, lane);
  __syncthreads();
  store_values<float, NL>(lds + (w * 64 + lane) * NL, gA);
  float* more = lds + W * 64 * NL;
  if (q == 0) more[w * 64 + c] = gD, more[(W + w) * 64 + c] = gbias;
  __syncthreads();
  if (w > 0 || !on) return;
  for (int o = 1; o < W; ++o) {
    float v[NL];
    load_values<float, NL>(lds + (o * 64 + lane) * NL, v);
#pragma unroll
    for (int j = 0; j < NL; ++j) gA[j] += v[j];
    gD += more[o * 64 + c], gbias += more[(W + o) * 64 + c];
  }
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const long at = ((long)b * p.channels + ch) * p.N + q * NL + j;
    if (q * NL + j < p.N) {
      p.a_part[at] = gA[j];
      if (p.gstate) p.gstate[at] = R[j];
    }
  }
  if (q == 0) p.d_part[(long)b * p.channels + ch] = gD, p.bias_part[(long)b * p.channels + ch] = gbias;
}

int scan_bwd(const ScanArgs& p, const ScanPlan& plan, int dtype, hipStream_t stream) {
  const unsigned grid = (unsigned)((long)plan.blocks * p.G * p.batch);
  const int CW = 64 / plan.NS, floats = plan.W * (2 * 16 * plan.NS * plan.NL + 3 * CW * 20 + 2 * 3 * 64 * plan.NL);
  const size_t lds = sizeof(float) * (size_t)floats;
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
