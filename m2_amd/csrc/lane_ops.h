// What the causal mixer's kernels (causal_conv_kernels.hip, selective_scan_kernels.hip, group_norm_kernels.hip) share: vectors of fp32 or bf16 values in memory,
// sums across lanes, sigmoid, softplus, and the sum over partial gradients.
#pragma once
#include "m2_internal.h"

namespace m2 {

// V consecutive values of a type in memory (float, or uint16_t: bf16) as floats; the address is a multiple of their size (V a power of two, up to 16 bytes).
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* p, float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 1) {
      f[0] = *p;
    } else {
      typedef float vec __attribute__((ext_vector_type(V)));
      const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = v[i];
    }
  } else if constexpr (V == 1) {
    f[0] = bf16_to_f32(*p);
  } else {
    typedef uint32_t vec __attribute__((ext_vector_type(V / 2 > 1 ? V / 2 : 2)));
    uint32_t w[V / 2];
    if constexpr (V == 2) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = v[i];
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_values(T* p, const float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 1) {
      *p = f[0];
    } else {
      typedef float vec __attribute__((ext_vector_type(V)));
      vec v;
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = f[i];
      *reinterpret_cast<vec*>(p) = v;
    }
  } else if constexpr (V == 1) {
    *p = f32_to_bf16(f[0]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(f[0], f[1]);
  } else {
    typedef uint32_t vec __attribute__((ext_vector_type(V / 2)));
    vec v;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<vec*>(p) = v;
  }
}

// What one lane of a wave has put into LDS is there for the others: orders the compiler's accesses, the hardware keeps a wave's own in order.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// What v holds in the lane whose number differs in bit BIT, for lanes that have that bit 0 (HIGH false) or 1.
template <int BIT, bool HIGH>
__device__ __forceinline__ float from_partner(float v) {
  if constexpr (BIT == 0) return dpp<0xB1>(v);                      // quad_perm 1 0 3 2
  else if constexpr (BIT == 1) return dpp<0x4E>(v);                 // quad_perm 2 3 0 1
  else if constexpr (BIT == 2) return HIGH ? dpp<0x124>(v) : dpp<0x12C>(v);      // row_ror 4, 12
  else return dpp<0x128>(v);                                        // row_ror 8
}
// v summed over the lanes that differ in bit BIT alone.
template <int BIT>
__device__ __forceinline__ float sum_over_bit(float v, int lane) {
  if constexpr (BIT >= 4) {
    const uint32_t u = __float_as_uint(v);
    const auto s = BIT == 5 ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
  } else if constexpr (BIT == 2) {
    const float low = from_partner<2, false>(v), high = from_partner<2, true>(v);      // (by all lanes, ahead of the choice)
    return v + (lane & 4 ? high : low);
  } else {
    return v + from_partner<BIT, false>(v);
  }
}
// Sums over the lanes that differ in bit BIT alone: of `zero` for lanes that have the bit 0, of `one` for the others.
template <int BIT>
__device__ __forceinline__ float split_over_bit(float zero, float one, int lane) {
  if constexpr (BIT >= 4) {
    const uint32_t a = __float_as_uint(zero), b = __float_as_uint(one);
    // rows (16: of 16 lanes, 32: halves) of one operand change places with those of the other, so that each lane has both values of its own sum
    const auto s = BIT == 5 ? __builtin_amdgcn_permlane32_swap(a, b, false, false) : __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
  } else {
    const float low = zero + from_partner<BIT, false>(zero), high = one + from_partner<BIT, true>(one);
    return (lane >> BIT) & 1 ? high : low;
  }
}
// v summed over groups of P (a power of two) neighbouring lanes.
template <int P>
__device__ __forceinline__ float lane_sum(float v, int lane) {
  if constexpr (P > 1) v = sum_over_bit<0>(v, lane);
  if constexpr (P > 2) v = sum_over_bit<1>(v, lane);
  if constexpr (P > 4) v += dpp<0x141>(v);      // row_half_mirror: quads hold one value by now
  if constexpr (P > 8) v += dpp<0x140>(v);      // row_mirror
  if constexpr (P > 16) v = sum_over_bit<4>(v, lane);
  if constexpr (P > 32) v = sum_over_bit<5>(v, lane);
  return v;
}

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// exp(x), x <= 88, to about 2^-23 of itself: the product with log2 e in two parts, of which the second is a factor near 1 (1.925963033500e-8 is log2 e less its fp32 rounding, kLog2E).  Below -100: as
// at -100 (NaN too).
__device__ __forceinline__ float exp_of(float x) {
  x = fmaxf(x, -100.f);
  const float hi = x * kLog2E;
  const float lo = fmaf(x, 1.925963033500e-8f, fmaf(x, kLog2E, -hi));      // what hi has lost, and log2 e beyond its 24 bits
  const float e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e, lo * kLn2, e);
}
// x / (1 + exp(-x)) among values of type T: with bf16 the exponential has its argument as it is rounded (off by |x| 2^-23 of itself at most, against the 2^-8 of a bf16 value), which saves six of
// eleven instructions.  The same goes for the slopes below, which also are factors of fp32 results (with bf16 hidden states: the gradients of the convolution's and group norm's weights and biases, and of
// a gated scan's A, D, dt_bias and state): each of their terms is off by |x| 2^-23 of itself more, a fraction of what the bf16 value in it was rounded by.
template <typename T>
__device__ __forceinline__ float silu(float x) {
  const float e = sizeof(T) == 2 ? __builtin_amdgcn_exp2f(x * -kLog2E) : exp_of(fminf(-x, 88.f));
  return x * __builtin_amdgcn_rcpf(1.f + e);
}
// u = exp(-|x|) and r = 1 / (1 + u): what sigmoid(x), sigmoid(-x), softplus(x) and their products are made of, without cancellation.
// EXACT: the exponential to 2^-23 of itself; else, for bf16 hidden states, as in silu.
template <bool EXACT>
struct Logistic {
  float u, r;
  bool below;
  __device__ __forceinline__ explicit Logistic(float x) : u(EXACT ? exp_of(-fabsf(x)) : __builtin_amdgcn_exp2f(-kLog2E * fabsf(x))), r(__builtin_amdgcn_rcpf(1.f + u)), below(x < 0.f) {}
  __device__ __forceinline__ float value() const { return below ? u * r : r; }
  __device__ __forceinline__ float other() const { return below ? r : u * r; }      // of -x
};
// log(1 + exp(x)) = max(x, 0) + log(1 + u), u = exp(-|x|) <= 1: log(w) of the rounded w = 1 + u, and what the rounding has lost over w (1 / w by a parabola: 6 % are enough).
__device__ __forceinline__ float softplus_of(float x, float u) {
  const float w = 1.f + u, lost = u - (w - 1.f);
  const float l = fmaf(__builtin_amdgcn_logf(w), kLn2, lost * fmaf(u, fmaf(u, 0.5f, -1.f), 1.f));
  return (x < 0.f ? 0.f : x) + l;
}
__device__ __forceinline__ float softplus(float x) { return softplus_of(x, exp_of(-fabsf(x))); }
// d/dx of x sigmoid(x) = s + x s (1 - s)
template <bool EXACT>
__device__ __forceinline__ float silu_slope_of(float x, const Logistic<EXACT>& l) {
  const float s = l.value();
  return fmaf(s * x, l.other(), s);
}
template <typename T>
__device__ __forceinline__ float silu_slope(float x) { return silu_slope_of(x, Logistic<sizeof(T) == 4>(x)); }

// Workgroups go round the eight XCDs: those of neighbouring numbers after this share one and its L2.
__device__ __forceinline__ int xcd_order(int id, int count) {
  const int each = count / 8, rest = count % 8, x = id % 8;
  return id / 8 + x * each + min(x, rest);
}

// Sums of `rows` partial results: column j of plane k (planes (K + 1 or 1) x n values) goes to wide[j * K + k] for k < K and to last[j] for k = K; either may be null.
int sum_partials(const float* partials, long rows, int K, long n, float* wide, float* last, hipStream_t stream);

}  // namespace m2
