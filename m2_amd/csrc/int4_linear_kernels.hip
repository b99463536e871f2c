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

constexpr int kRows = 4;

// A wave has a tile's 16 rows of W and up to four of x; its lanes share K.
template <typename T, int GROUP>
__global__ __launch_bounds__(256) void int4_linear_kernel(const T* __restrict__ x, long x_row, const unsigned char* __restrict__ w,
                                                          const float* __restrict__ bias, T* __restrict__ out, int M, int N, int K, int gelu) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = (int)blockIdx.x * 4 + wave, m0 = (int)blockIdx.y * kRows, kt = (K + kTileK - 1) / kTileK;
  if (tile * kTileN >= N) return;
  float acc[kRows] = {};
  for (int b = 0; b < kt; ++b) {
    const unsigned char* p = w + ((long)tile * kt + b) * tile_bytes(GROUP);
    const uint4 q4 = *reinterpret_cast<const uint4*>(p + lane * 16);
    const uint32_t q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      const float s = bf16_to_f32(*reinterpret_cast<const uint16_t*>(p + 1024 + ((lane & 15) * (kTileK / GROUP) + step * 32 / GROUP) * 2));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = b * kTileK + step * 32 + (lane >> 4) * 8 + j;
        const float v = (float)((int)((q[step] >> (16 * (j % 2) + 4 * (j / 2))) & 15) - 8) * s;
        if (k < K)
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const T* row = x + (long)min(m0 + r, M - 1) * x_row;
            float xv;
            if constexpr (sizeof(T) == 4) xv = row[k]; else xv = bf16_to_f32(row[k]);
            acc[r] = fmaf(xv, v, acc[r]);
          }
      }
    }
  }
  const int n = tile * kTileN + (lane & 15);
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float y = acc[r];
    y += __shfl_xor(y, 16);
    y += __shfl_xor(y, 32);
    if (lane < 16 && n < N && m0 + r < M) {
      y += bias ? bias[n] : 0.f;
      if (gelu) y = gelu_erf(y);
      if constexpr (sizeof(T) == 4) out[(long)(m0 + r) * N + n] = y; else out[(long)(m0 + r) * N + n] = f32_to_bf16(y);
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
  const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + kRows - 1) / kRows));
  const auto go = [&](auto kernel, auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, (const T*)x, x_row, (const unsigned char*)weight, bias, (T*)out, M, N, K, gelu);
  };
  const auto pick = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (group == 32) go(int4_linear_kernel<T, 32>, t);
    else if (group == 64) go(int4_linear_kernel<T, 64>, t);
    else go(int4_linear_kernel<T, 128>, t);
  };
  dtype == M2_DTYPE_F32 ? pick((float*)nullptr) : pick((uint16_t*)nullptr);
  return check_launch("int4_linear");
}
