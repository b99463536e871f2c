// y = act(x W^T + b) for few rows x, W (N, K) in 4 bits with a bf16 scale for each group of a row: W[n, k] = (q - 8) s, q in 0 .. 15.
//
// What bounds it is the weight: N K / 2 bytes for a few rows of sums.
//
// Order of the weights in memory: tiles of 16 rows n by 128 columns k, those of the same rows behind one another.  A tile is 64 lanes times 16 bytes, lane l
// = 16 (k / 8 % 4) + n % 16 with the eight k of each of the four steps of 32 in a 32-bit word, value j of the eight at bit 16 (j % 2) + 4 (j / 2); behind them
// 16 rows times 128 / group scales.  K and N are padded with q = 8 and scale 0.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "m2_internal.h"

namespace m2 {

constexpr int kTileK = 128, kTileN = 16;

constexpr int tile_bytes(int group) { return 64 * 16 + kTileN * (kTileK / group) * 2; }

__device__ __forceinline__ float gelu_erf(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f)); }

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) u32x4_any;      // at any address of x's type

// Eight codes as bf16 16 + q, exactly: 0x4180 is 16, and its last bits but three are worth 1 each.  What a row of x sums to, times 24, is taken off again.
__device__ __forceinline__ bf16x8 codes(uint32_t q) {
  const u32x4 v = {((q << 3) & 0x00780078u) | 0x41804180u, ((q >> 1) & 0x00780078u) | 0x41804180u, ((q >> 5) & 0x00780078u) | 0x41804180u,
                   ((q >> 9) & 0x00780078u) | 0x41804180u};
  return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ bf16x8 minus24() {
  const u32x4 v = {0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u};
  return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Rows of x as the operand of 16 rows by 32 columns: lane l has row l % 16, columns 8 (l / 16) .. + 7.
// bf16: 16 rows.  fp32: 4 rows in 4 places each, the first three of them the row's three bf16 parts, x = part + part + part with the low bits
// cut off in turn (no rounding, so none overflows); what the fourth holds is not looked at.
template <typename T> struct Operand;
template <> struct Operand<uint16_t> {
  static constexpr int kRows = 16;
  static __device__ __forceinline__ int row(int lane) { return lane & 15; }
  u32x4 v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = *reinterpret_cast<const u32x4_any*>(p); }
  __device__ __forceinline__ void one(const uint16_t* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (2 * i < n ? p[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)p[2 * i + 1] << 16 : 0u);
  }
  __device__ __forceinline__ void keep(bool is) { v = is ? v : u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ bf16x8 get(int) const { return __builtin_bit_cast(bf16x8, v); }
};
template <> struct Operand<float> {
  static constexpr int kRows = 4;
  static __device__ __forceinline__ int row(int lane) { return (lane & 15) >> 2; }
  u32x4 v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = *reinterpret_cast<const u32x4_any*>(p);
    v[1] = *reinterpret_cast<const u32x4_any*>(p + 4);
  }
  __device__ __forceinline__ void one(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = i < n ? __float_as_uint(p[i]) : 0u;
  }
  __device__ __forceinline__ void keep(bool is) { v[0] = is ? v[0] : u32x4{0, 0, 0, 0}, v[1] = is ? v[1] : u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ bf16x8 get(int lane) const {
    const uint32_t second = (lane & 3) > 0 ? 0xffff0000u : 0u, third = (lane & 3) > 1 ? 0xffff0000u : 0u;
    uint32_t f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = __uint_as_float(v[i / 4][i % 4]);
      x -= __uint_as_float(__float_as_uint(x) & second);
      x -= __uint_as_float(__float_as_uint(x) & third);
      f[i] = __float_as_uint(x);
    }
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_perm(f[2 * i + 1], f[2 * i], 0x07060302u);      // the upper halves
    return __builtin_bit_cast(bf16x8, o);
  }
};

// The eight values of a row from column k on, 0 behind the last: where K is a multiple of eight (EVEN), all of them or none; else one by one.
template <typename T, bool EVEN>
__device__ __forceinline__ void load_edge(Operand<T>& to, const T* row, int k, int K) {
  if (EVEN) {
    to.load(row + (k < K ? k : 0));
    to.keep(k < K);
  } else {
    to.one(row + k, K - k);
  }
}

// The scales of a lane's row in a tile.
template <int GROUP>
struct Scales {
  uint32_t v[GROUP == 32 ? 2 : 1];
  __device__ __forceinline__ void load(const unsigned char* tile, int lane) {
    const unsigned char* p = tile + 1024 + (lane & 15) * (kTileK / GROUP) * 2;
    if (GROUP == 32) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      v[0] = u.x;
      v[GROUP == 32 ? 1 : 0] = u.y;
    } else {
      v[0] = GROUP == 64 ? *reinterpret_cast<const uint32_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float get(int g) const { return __uint_as_float(g % 2 ? v[g / 2] & 0xffff0000u : v[g / 2] << 16); }
};

// 128 columns of x's rows and of NT tiles of W: what a wave has asked for, and what it makes of it.
template <typename T, int GROUP, bool EVEN, int NT>
struct Step {
  u32x4 q[NT];
  Scales<GROUP> s[NT];
  Operand<T> x[4];
  // `w`: the first tile's part, the others' `apart` bytes behind one another; those from `tiles` on are the last one again
  __device__ __forceinline__ void load(const unsigned char* w, long apart, int tiles, const T* row, int b, int K, int lane) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const unsigned char* p = w + min(t, tiles - 1) * apart + (long)b * tile_bytes(GROUP);
      q[t] = *reinterpret_cast<const u32x4*>(p + lane * 16);
      s[t].load(p, lane);
    }
    const int k = b * kTileK + (lane >> 4) * 8;
    if ((b + 1) * kTileK <= K) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i].load(row + k + i * 32);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_edge<T, EVEN>(x[i], row, k + i * 32, K);
    }
  }
  __device__ __forceinline__ void add(floatx4 (&sum)[NT], int lane) const {
    constexpr int kSteps = GROUP / 32;
#pragma unroll
    for (int g = 0; g < kTileK / GROUP; ++g) {
      bf16x8 a[kSteps];
      floatx4 c0 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        a[i] = x[g * kSteps + i].get(lane);
        c0 = mfma(a[i], minus24(), c0);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        floatx4 c = c0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) c = mfma(a[i], codes(q[t][g * kSteps + i]), c);
        const float scale = s[t].get(g);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[t][i] = fmaf(scale, c[i], sum[t][i]);
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void put(T* out, long at, float y, int gelu) {
  if (gelu) y = gelu_erf(y);
  if constexpr (sizeof(T) == 4) out[at] = y; else out[at] = f32_to_bf16(y);
}

constexpr int waves_of(int split) { return split > 4 ? split : 4; }

// Up to 16 rows of bf16 or 4 of fp32.  A wave has NT tiles of 16 rows of W, and of their tiles of 128 columns every SPLIT-th; the SPLIT waves' sums meet in shared
// memory.
template <typename T, int GROUP, bool EVEN, int NT, int SPLIT>
__global__ __launch_bounds__(64 * waves_of(SPLIT)) void int4_few_rows_kernel(const T* __restrict__ x, long x_row, const unsigned char* __restrict__ w, const float* __restrict__ bias,
                                                            T* __restrict__ out, int M, int N, int K, int gelu) {
  __shared__ floatx4 sums[SPLIT > 1 ? waves_of(SPLIT) : 1][SPLIT > 1 ? NT : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (N + kTileN - 1) / kTileN, kt = (K + kTileK - 1) / kTileK;
  const int t0 = ((int)blockIdx.x * (waves_of(SPLIT) / SPLIT) + wave / SPLIT) * NT, part = wave % SPLIT, m0 = (int)blockIdx.y * Operand<T>::kRows;
  floatx4 sum[NT] = {};
  if (t0 < tiles) {
    const long apart = (long)kt * tile_bytes(GROUP);
    const unsigned char* mine = w + t0 * apart;
    const T* row = x + (long)min(m0 + Operand<T>::row(lane), M - 1) * x_row;
    Step<T, GROUP, EVEN, NT> now, next;
    if (part < kt) now.load(mine, apart, tiles - t0, row, part, K, lane);
    for (int b = part; b < kt; b += SPLIT) {
      if (b + SPLIT < kt) next.load(mine, apart, tiles - t0, row, b + SPLIT, K, lane);
      now.add(sum, lane);
      now = next;
    }
  }
  if (SPLIT > 1) {
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[wave][t][lane] = sum[t];
    __syncthreads();
    if (NT == 1 && part) return;
  }
  // with more than one tile the waves share them out
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (SPLIT > 1) {
      if (NT > 1 && t % SPLIT != part) continue;
      sum[t] = sums[wave - part][t][lane];
#pragma unroll
      for (int i = 1; i < SPLIT; ++i) sum[t] += sums[wave - part + i][t][lane];
    }
    const int n = (t0 + t) * kTileN + (lane & 15);
    if (n >= N) continue;
    const float b = bias ? bias[n] : 0.f;
    if constexpr (sizeof(T) == 4) {
      const int m = m0 + (lane >> 4);
      if (m < M) put(out, (long)m * N + n, (sum[t][2] + sum[t][1]) + sum[t][0] + b, gelu);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + (lane >> 4) * 4 + i;
        if (m < M) put(out, (long)m * N + n, sum[t][i] + b, gelu);
      }
    }
  }
}

// More rows: a workgroup has MT times 16 places of rows (as Operand) and 4 NT tiles of W's rows, NT a wave.  x goes through shared memory, one tile of 128
// columns after the other in two buffers, in the operand's order: 64 lanes times 16 bytes for each 16 places and 32 columns.  A lane's place among
// the 16 of its eighth is turned by the number of the eighth, so that the threads that write a row's sixteen eighths meet in no bank; readers are permuted
// among themselves.
template <typename T, bool EVEN, int MT>
struct Staged {
  static constexpr int kRows = MT * Operand<T>::kRows, kBytes = MT * 4 * 1024, kEach = kRows / 16;      // kEach: eighths of a thread
  static_assert(kRows % 16 == 0, "a row for every 16 threads");
  Operand<T> v[kEach];
  __device__ __forceinline__ void load(const T* x, long x_row, int m0, int M, int b, int K) {
    const int k = b * kTileK + (threadIdx.x & 15) * 8;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const T* row = x + (long)min(m0 + (int)(threadIdx.x >> 4) + 16 * i, M - 1) * x_row;
      if ((b + 1) * kTileK <= K) v[i].load(row + k); else load_edge<T, EVEN>(v[i], row, k, K);
    }
  }
  __device__ __forceinline__ void store(unsigned char* to) const {
    const int c = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int row = (int)(threadIdx.x >> 4) + 16 * i;
      constexpr int kPlaces = sizeof(T) == 4 ? 3 : 1, kSpread = sizeof(T) == 4 ? 4 : 1;
#pragma unroll
      for (int part = 0; part < kPlaces; ++part) {
        const int place = row * kSpread + part;
        *reinterpret_cast<bf16x8*>(to + (place / 16 * 4 + c / 4) * 1024 + (c % 4 * 16 + ((place & 15) ^ c)) * 16) = v[i].get(part);
      }
    }
  }
  static __device__ __forceinline__ bf16x8 read(const unsigned char* from, int mt, int step, int lane) {
    const int c = step * 4 + (lane >> 4);
    return *reinterpret_cast<const bf16x8*>(from + (mt * 4 + step) * 1024 + ((lane & 48) + ((lane & 15) ^ c)) * 16);
  }
};

template <typename T, int GROUP, bool EVEN, int MT, int NT>
__global__ __launch_bounds__(256, 2) void int4_rows_kernel(const T* __restrict__ x, long x_row, const unsigned char* __restrict__ w, const float* __restrict__ bias,
                                                        T* __restrict__ out, int M, int N, int K, int gelu, int row_blocks) {
  constexpr int kSteps = GROUP / 32;
  __shared__ __attribute__((aligned(16))) unsigned char staged[2][Staged<T, EVEN, MT>::kBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (N + kTileN - 1) / kTileN, kt = (K + kTileK - 1) / kTileK;
  const int m0 = (int)(blockIdx.x % row_blocks) * Staged<T, EVEN, MT>::kRows, t0 = ((int)(blockIdx.x / row_blocks) * 4 + wave) * NT;
  const unsigned char* mine[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) mine[t] = w + (long)min(t0 + t, tiles - 1) * kt * tile_bytes(GROUP);
  floatx4 sum[MT][NT] = {};
  Staged<T, EVEN, MT> x_now;
  u32x4 q[NT], q_next[NT];
  Scales<GROUP> s[NT], s_next[NT];
  const auto ask = [&](int b) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const unsigned char* p = mine[t] + (long)b * tile_bytes(GROUP);
      q_next[t] = *reinterpret_cast<const u32x4*>(p + lane * 16);
      s_next[t].load(p, lane);
    }
    x_now.load(x, x_row, m0, M, b, K);
  };
  ask(0);
  x_now.store(staged[0]);
  __syncthreads();
  for (int b = 0; b < kt; ++b) {
#pragma unroll
    for (int t = 0; t < NT; ++t) q[t] = q_next[t], s[t] = s_next[t];
    if (b + 1 < kt) ask(b + 1);
    const unsigned char* from = staged[b & 1];
#pragma unroll
    for (int g = 0; g < kTileK / GROUP; ++g) {
      bf16x8 a[MT][kSteps];
      floatx4 c0[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        c0[m] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          a[m][i] = Staged<T, EVEN, MT>::read(from, m, g * kSteps + i, lane);
          c0[m] = mfma(a[m][i], minus24(), c0[m]);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bf16x8 v[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) v[i] = codes(q[t][g * kSteps + i]);
        const float scale = s[t].get(g);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          floatx4 c = c0[m];
#pragma unroll
          for (int i = 0; i < kSteps; ++i) c = mfma(a[m][i], v[i], c);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[m][t][i] = fmaf(scale, c[i], sum[m][t][i]);
        }
      }
    }
    if (b + 1 < kt) x_now.store(staged[(b + 1) & 1]);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = (t0 + t) * kTileN + (lane & 15);
    if (n >= N) continue;
    const float bn = bias ? bias[n] : 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (sizeof(T) == 4) {
        const int row = m0 + m * 4 + (lane >> 4);
        if (row < M) put(out, (long)row * N + n, (sum[m][t][2] + sum[m][t][1]) + sum[m][t][0] + bn, gelu);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = m0 + m * 16 + (lane >> 4) * 4 + i;
          if (row < M) put(out, (long)row * N + n, sum[m][t][i] + bn, gelu);
        }
      }
    }
  }
}

}  // namespace m2

using namespace m2;

extern "C" size_t m2_int4_weight_bytes(int N, int K, int group) {
  if (N <= 0 || K <= 0 || (group != 32 && group != 64 && group != 128)) return 0;
  return (size_t)((N + kTileN - 1L) / kTileN) * (size_t)((K + kTileK - 1L) / kTileK) * (size_t)tile_bytes(group);
}

extern "C" int m2_int4_linear_fwd(const void* x, long x_row, const void* weight, const float* bias, void* out, int M, int N, int K, int group, int gelu,
                                  int dtype, void* stream) {
  const char* who = "m2_int4_linear_fwd";
  if (!x || !weight || !out) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype must be M2_DTYPE_F32 or M2_DTYPE_BF16 (got %d)", who, dtype);
  if (M <= 0 || N <= 0 || K <= 0 || x_row < 0 || (gelu != 0 && gelu != 1)) return set_error(M2_ERR_ARG, "%s: M=%d N=%d K=%d x_row=%ld gelu=%d", who, M, N, K, x_row, gelu);
  if (group != 32 && group != 64 && group != 128) return set_error(M2_ERR_UNSUPPORTED, "%s: groups of 32, 64 or 128 values (got %d)", who, group);
  if (!aligned16(weight)) return set_error(M2_ERR_UNSUPPORTED, "%s: the weight must be 16-byte aligned", who);
  const uintptr_t size = dtype == M2_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)x % size || (uintptr_t)out % size || (uintptr_t)bias % 4) return set_error(M2_ERR_UNSUPPORTED, "%s: x, out and bias must be aligned to their type", who);
  hipStream_t st = (hipStream_t)stream;
  const int tiles = (N + kTileN - 1) / kTileN, kt = (K + kTileK - 1) / kTileK;
  const auto go = [&](auto kernel, auto* t, int nt, int split) {
    using T = std::remove_pointer_t<decltype(t)>;
    const long waves = (tiles + nt - 1L) / nt * split, each = waves_of(split);
    hipLaunchKernelGGL(kernel, dim3((unsigned)((waves + each - 1) / each), (unsigned)((M + Operand<T>::kRows - 1) / Operand<T>::kRows)), dim3(64 * each), 0, st, (const T*)x, x_row,
                       (const unsigned char*)weight, bias, (T*)out, M, N, K, gelu);
  };
  const auto rows = [&](auto kernel, auto* t, int mt, int nt) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int each = mt * Operand<T>::kRows, row_blocks = (M + each - 1) / each;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((tiles + 4L * nt - 1) / (4 * nt) * row_blocks)), dim3(256), 0, st, (const T*)x, x_row, (const unsigned char*)weight, bias,
                       (T*)out, M, N, K, gelu, row_blocks);
  };
  const auto parts = [&](auto* t, auto g) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int G = decltype(g)::value;
    const int places = (M + Operand<T>::kRows - 1) / Operand<T>::kRows;      // times 16
    if (places > 1) {
      constexpr int kMt = sizeof(T) == 4 ? 4 : 2;      // 32 rows of bf16, 16 of fp32
      const long blocks = (places + kMt - 1L) / kMt * ((tiles + 7) / 8);
      if (K % 8) return rows(int4_rows_kernel<T, G, false, kMt, 1>, t, kMt, 1);
      if (blocks < 512) return rows(int4_rows_kernel<T, G, true, kMt, 1>, t, kMt, 1);
      return rows(int4_rows_kernel<T, G, true, kMt, 2>, t, kMt, 2);
    }
    // Few tiles: all of a workgroup's waves share one.  More: tiles share what a wave reads (and splits) of x, four where that is as much as a tile, and
    // long rows are shared by eight waves.  us, NT and SPLIT 1, 8 / 2, 4 / 2, 8 / 4, 4 / 4, 8: 768 -> 768 M = 1 2.7 / 3.3 / 3.2 / 4.2 / 3.8; 4096 -> 4096 M = 16
    // 7.2 / 8.7 / 7.5 / 11.7 / 9.4; 1792 -> 7168 M = 16 7.2 / 6.6 / 5.6 / 7.0 / 7.0; 768 -> 30528 M = 1 6.6 / 6.1 / 6.7 / 6.8 / 6.5, M = 16 9.3 / 7.0 / 7.4 / 6.9 / 6.9;
    // 4096 -> 16384 M = 1 10.0 / 10.3 / 9.4 / 12.4 / 9.9, M = 16 19.5 / 13.0 / 13.0 / 13.4 / 11.2; 7168 -> 16384 fp32 M = 1 24.6 / 18.6 / 17.4 / 17.5 / 14.7.
    if (K % 8) return go(int4_few_rows_kernel<T, G, false, 1, 8>, t, 1, 8);
    if (tiles < 384) return go(int4_few_rows_kernel<T, G, true, 1, 8>, t, 1, 8);
    if (tiles >= 1024 && (sizeof(T) == 4 || M > 8))
      return kt < 16 ? go(int4_few_rows_kernel<T, G, true, 4, 4>, t, 4, 4) : go(int4_few_rows_kernel<T, G, true, 4, 8>, t, 4, 8);
    return kt < 16 ? go(int4_few_rows_kernel<T, G, true, 2, 4>, t, 2, 4) : go(int4_few_rows_kernel<T, G, true, 2, 8>, t, 2, 8);
  };
  const auto pick = [&](auto* t) {
    if (group == 32) parts(t, std::integral_constant<int, 32>{});
    else if (group == 64) parts(t, std::integral_constant<int, 64>{});
    else parts(t, std::integral_constant<int, 128>{});
  };
  dtype == M2_DTYPE_F32 ? pick((float*)nullptr) : pick((uint16_t*)nullptr);
  return check_launch("int4_linear");
}
