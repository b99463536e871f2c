// What the selective scan's kernels share: arguments, how a wave lies over channels, states and positions, and how its tiles come in.
#pragma once
#include <type_traits>

#include "lane_ops.h"

namespace m2 {

struct ScanArgs {
  // x, dt, z (B, L, D) and gy: a batch and a row apart; Bm, Cm (B, L, G, N): and a group apart
  const void *x, *dt, *z, *Bm, *Cm, *gy;
  long x_batch, x_row, dt_batch, dt_row, z_batch, z_row, b_batch, b_row, b_group, c_batch, c_row, c_group, gy_batch, gy_row;
  const float *A, *D, *dt_bias, *state;      // (D, N), (D), (D) and (B, D, N); the last three or null
  const long long* lengths;                  // (B) or null
  void* y;                                   // (B, L, D)
  float* state_out;                          // (B, D, N) or null
  float* saved;                              // (B, parts, D, N): the state ahead of each part of a sequence, for the gradient, or null
  int batch, L, channels, G, N, softplus;
  int per_group, blocks, parts;              // channels of a group, workgroups for them, parts of a sequence
  int apart;                                 // positions between the states that are kept: a step of the gradient's workgroups
  int sets;                                  // the gradient: sets of 64 / NS channels that a workgroup takes one after the other
  // gradients
  const float* gstate_out;                   // or null
  void *gx, *gdt, *gz;                       // (B, L, D)
  float* gstate;                             // (B, D, N) or null
  float *b_part, *c_part;                    // (blocks, B, L, G, N)
  float *a_part, *d_part, *bias_part;        // (B, D, N), (B, D), (B, D)
};

// The kernel's arguments anew: values that are read where they are needed, and not kept in (too few) scalar registers from the kernel's start.
typedef const __attribute__((address_space(4))) ScanArgs ArgsInMemory;
__device__ __forceinline__ ArgsInMemory* arguments_anew() {
  ArgsInMemory* p = (ArgsInMemory*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// A wave takes 64 / NS channels times NS lanes with NL states each, for TT positions.  QLOW: a channel's lanes are neighbours; else they lie 64 / NS apart.
template <int NS, int NL>
struct ScanShape {
  static constexpr int CW = 64 / NS, NP = NS * NL, TT = 16;
  static constexpr int NT = NS < TT ? TT / NS : 1;      // positions whose x, dt, z and y a lane moves: q, q + NS, ...
  static constexpr int PITCH = TT + 4;                  // of a channel's positions in shared memory: 16-byte reads of neighbouring channels hit different banks
  static constexpr int TILE = TT * NP;                  // B or C of the positions
  static constexpr int NB = TILE / 4 / 64 > 1 ? TILE / 4 / 64 : 1;      // vectors of four of it that a lane moves
  static constexpr bool AHEAD = NB <= 4;
};
constexpr int log2_of(int n) { return n > 1 ? 1 + log2_of(n / 2) : 0; }

__device__ __forceinline__ int scan_length(const ScanArgs& p, int b) {
  if (!p.lengths) return p.L;
  const long long n = p.lengths[b];
  return n < 0 ? 0 : n > p.L ? p.L : (int)n;
}

// Four values of a row of B or C as they are in memory, at any address of their type.
template <typename T> struct Raw4;
template <> struct Raw4<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ float get(const type& v, int i) { return v[i]; }
};
template <> struct Raw4<uint16_t> {
  typedef uint16_t type __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ float get(const type& v, int i) { return bf16_to_f32(v[i]); }
};
template <typename T>
__device__ __forceinline__ float value_of(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return bf16_to_f32(v);
}
template <typename T>
__device__ __forceinline__ T value_to(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else return f32_to_bf16(v);
}

// The value is made here: one made of a loaded register only later would hold that register over the next load into it, which a loop then waits for.
__device__ __forceinline__ void made_here(float& v) { asm volatile("" : "+v"(v)); }

// A in powers of two, kept within fp32's range: the positions behind an end have a step of 0, and 0 times an infinity would leave them a state that is no number.
__device__ __forceinline__ float decay_rate(float A) {
  constexpr float kMost = 3.402823466e38f;
  const float r = A * kLog2E;
  return r < -kMost ? -kMost : r > kMost ? kMost : r;      // (NaN stays)
}

// A value at a byte offset from what is the same for all lanes: a scalar address and a 32-bit offset.
template <typename V, typename T>
__device__ __forceinline__ V& at_offset(T* base, uint32_t bytes) {
  if constexpr (std::is_const<T>::value) return *reinterpret_cast<V*>(reinterpret_cast<const char*>(base) + bytes);
  else return *reinterpret_cast<V*>(reinterpret_cast<char*>(base) + bytes);
}

// Where a lane's values of a tensor (rows `row` values apart, below 2^24) lie from row t0 of it, in bytes: those of row t0 + t, but of no row behind `last`.  Rows
// grow with offsets, so the smaller offset is the nearer row; one load serves both, and nothing waits for a choice.
struct Near {
  uint32_t first, end;
  template <typename T>
  __device__ __forceinline__ static Near of(const T*, int t, long row, int at, int last) {
    // (a product of 24-bit factors takes a quarter of the time)
    return {(__umul24((uint32_t)t, (uint32_t)row) + (uint32_t)at) * (uint32_t)sizeof(T), (uint32_t)(last * (int)row + at) * (uint32_t)sizeof(T)};
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t further) const { return min(first + further, end); }
};

// B or C of a wave's positions on their way from memory (positions t0 .. of a sequence of n > t0; beyond it, the last one's are read) to fp32 in shared memory,
// (TT, NP), zero behind N.
template <typename T, int NS, int NL, int COUNT>
struct TileIn {
  using S = ScanShape<NS, NL>;
  static constexpr int PER = S::NP >= 4 ? S::NP / 4 : 1, APART = 64 / PER > 1 ? 64 / PER : 1;      // vectors of a row; rows between a lane's vectors
  typename Raw4<T>::type raw[COUNT];
  __device__ __forceinline__ void load(const T* rows, long row, int t0, int n, int N, int lane, int first = 0) {
    const T* base = rows + (long)t0 * row;
    const int last = min(n - 1 - t0, S::TT - 1);
    if constexpr (S::NP >= 4) {
      if (N >= 4) {      // a vector that would pass N ends with it
        const Near off = Near::of(rows, min(lane / PER, S::TT - 1), row, min(lane % PER * 4, N - 4), last);
#pragma unroll
        for (int i = 0; i < COUNT; ++i) raw[i] = at_offset<const typename Raw4<T>::type>(base, off((uint32_t)((first + i) * APART * (int)row) * (uint32_t)sizeof(T)));
      } else {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
          const T* r = base + (long)min(min(lane / PER, S::TT - 1) + (first + i) * APART, last) * row;
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[i][j] = j < N ? r[j] : T(0);
        }
      }
    } else {
      const int at = lane % S::NP;
      raw[0][0] = at < N ? base[(long)min(lane / S::NP, last) * row + at] : T(0);
    }
  }
  __device__ __forceinline__ void put(float* tile, int N, int lane, int first = 0) const {
    if constexpr (S::NP >= 4) {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        const int v = lane + 64 * (first + i), at = lane % PER * 4;
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = Raw4<T>::get(raw[i], j);
        if (N >= 4 && N < S::NP) {      // (the same for all lanes)
          float g[4];
          const int moved = at - min(at, N - 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g[j] = 0.f;
#pragma unroll
            for (int k = j; k < 4; ++k) g[j] = k - j == moved ? f[k] : g[j];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = g[j];
        }
        if (v < S::TILE / 4) store_values<float, 4>(tile + v * 4, f);
      }
    } else if (lane < S::TILE) {
      tile[lane] = Raw4<T>::get(raw[0], 0);
    }
  }
};
template <typename T, int NS, int NL>
__device__ __forceinline__ void tile_in(float* tile, const T* rows, long row, int t0, int n, int N, int lane) {
  constexpr int NB = ScanShape<NS, NL>::NB, AT_ONCE = NB < 4 ? NB : 4;
  for (int first = 0; first < NB; first += AT_ONCE) {
    TileIn<T, NS, NL, AT_ONCE> in;
    in.load(rows, row, t0, n, N, lane, first);
    in.put(tile, N, lane, first);
  }
}

// Sums over the NS lanes of a channel of one value for each of TT positions (register t, in place): lane q keeps positions q, q + NS, ... as 0, 1, ...
// FIRST: lane bit of q's lowest bit.
template <int NS, int FIRST, int K = 0>
__device__ __forceinline__ void share_positions(float (&y)[16], int lane) {
  if constexpr ((1 << K) < NS) {
    constexpr int count = 16 >> K;
    if constexpr (count > 1) {
#pragma unroll
      for (int m = 0; m < count / 2; ++m) y[m] = split_over_bit<FIRST + K>(y[2 * m], y[2 * m + 1], lane);
    } else {
      y[0] = sum_over_bit<FIRST + K>(y[0], lane);
    }
    share_positions<NS, FIRST, K + 1>(y, lane);
  }
}

// f(NS, NL as constants), for the shapes that SERVED(NS, NL) says are built
template <typename SERVED, typename F>
void with_scan_shape(int NS, int NL, F&& f) {
  const auto with = [&](auto ns, auto nl) {
    if constexpr (SERVED::built(decltype(ns)::value, decltype(nl)::value)) f(ns, nl);
  };
  const auto with_lanes = [&](auto nl) {
    switch (NS) {
      case 1: return with(std::integral_constant<int, 1>{}, nl);
      case 2: return with(std::integral_constant<int, 2>{}, nl);
      case 4: return with(std::integral_constant<int, 4>{}, nl);
      case 8: return with(std::integral_constant<int, 8>{}, nl);
      case 16: return with(std::integral_constant<int, 16>{}, nl);
      case 32: return with(std::integral_constant<int, 32>{}, nl);
      default: return with(std::integral_constant<int, 64>{}, nl);
    }
  };
  if (NL == 1) with_lanes(std::integral_constant<int, 1>{});
  else if (NL == 2) with_lanes(std::integral_constant<int, 2>{});
  else with_lanes(std::integral_constant<int, 4>{});
}
// Those whose registers do not pass a wave's: four states of a lane hold 128 of decays and inputs, and many channels of a wave need more for each lane's own positions; the gradient has room
// for two, and for four only where no channels' sums are formed.
struct ForwardShapes {
  static constexpr bool built(int NS, int NL) { return NL <= 2 || NS >= 4; }
};
struct GradientShapes {
  static constexpr bool built(int NS, int NL) { return NL == 1 ? NS >= 2 : NL == 2 ? NS >= 4 : NS == 64; }
};

// How a call is spread: lanes a channel, states a lane, waves of a workgroup.
struct ScanPlan {
  int NS, NL, W, blocks, sets;
};

size_t scan_bwd_lds(const ScanPlan& plan);
int scan_bwd(const ScanArgs& p, const ScanPlan& plan, int dtype, hipStream_t stream);

}  // namespace m2
