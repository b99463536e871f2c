// y = act(x W^T + b) for few rows x, W (N, K) in 4 bits with a bf16 scale for each group of a row: W[n, k] = (q - 8) s, q in 0 .. 15.
//
// Few rows are bound by the weight, N K / 2 bytes and 2 N K / group of scales: 12.5 MB and 2.4 us for the word embeddings at K = 768, beside 3 us that any launch of
// a few dependent loads takes; a wave's loads, the 14 vector instructions for eight codes and the products stand behind one another (vector unit 38 % busy at 1 x 7168 -> 16384).  Many rows are
// bound by several things alike, which hardly overlap: of 34 us at M = 512 making W out of the codes takes 7, fetching x and W 7,
// the products 12 (as copies of the kernel without one or two of these say; the matrix unit is busy 27 % of the cycles, the vector unit 43 %), and workgroups twice as wide or high, 64 x 64
// instead of 64 x 32 to a wave, or another order of the instructions change nothing.  Kernel times, MI355X; beside them bytes at 5.3 TB/s or products at the 1.27 PFLOP/s that a large
// library product reaches (matrix instructions alone: 1.9):
//
//   M x K -> N              us (floor)             M x K -> N                  us (floor)
//   1 x 768 -> 30528        5.7 (2.4)              64 x 768 -> 30528           11.2 (3.1)
//   16 x 768 -> 30528       6.1 (2.6)              128 x 768 -> 30528          12.3 + 4.3 (4.7)
//   16 x 1001 -> 30522      8.6 (3.3)              512 x 768 -> 30528          34.6 + 4.4 (18.9)
//   13 x 1536 -> 30522      8.5 (4.7)              4096 x 1792 -> 1792         36.1 + 9.4 (20.7)
//   1 x 7168 -> 16384       12.7 (11.4)            40 x 768 -> 30522, fp32     10.6 + 4.2 (3.5)
//   16 x 7168 -> 16384      14.5 (11.6)            512 x 768 -> 30528, fp32    60 + 5.0 (37.8: two products of half-precision parts)
//   3 x 960 -> 960, fp32    3.5 (0.1)              8 x 5672 -> 1200, fp32      7.9 (0.7)
//   64 x 4096 -> 2000       8.6 (1.0)              512 x 7168 -> 1792          25.2 + 8.3 (10.4)
//
// A product runs on one of three kernels (plan_of): up to 16 rows of bf16 or 4 of fp32 straight from memory, and more of them so where W is small; more rows with x in shared
// memory; large products with x as half-precision operands, which a launch of its own writes (behind the +).
//
// Order of the weights in memory: tiles of 16 rows n by 128 columns k, those of the same rows behind one another.  A tile is 64 lanes times 16 bytes, lane l
// = 16 (k / 8 % 4) + n % 16 with the eight k of each of the four steps of 32 in a 32-bit word, value j of the eight at bit 16 (j % 2) + 4 (j / 2); behind them
// 16 rows times 128 / group scales.  K and N are padded with q = 8 and scale 0.  Behind all tiles a factor for each row, a power of two.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "m2_internal.h"
#include "mfma_stream.h"

namespace m2 {

constexpr int kTileK = 128, kTileN = 16;
constexpr int kMaxSize = 1 << 30;      // of N and K: what a workgroup's last tiles count to behind them stays below 2^31

constexpr int tile_bytes(int group) { return 64 * 16 + kTileN * (kTileK / group) * 2; }

__device__ __forceinline__ float gelu_erf(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f)); }

typedef uint32_t __attribute__((ext_vector_type(4), aligned(2))) u32x4_any;      // at any address of x's type
typedef uint32_t __attribute__((ext_vector_type(2), aligned(2))) u32x2_any;

// Eight codes as bf16 (q - 8) / 16, exactly; results are multiplied by 16 at the end.  The instruction takes the low four bits of a byte as a signed number to fp32, and q with its top bit turned
// is q - 8; the upper halves of two are put together.  Nothing has to be taken off a sum again, so that a value on a code of zero leaves it as it was.  16 + q, whose bits are quicker to make (8
// instructions instead of 14), less 24 times the sum of x kept 24 times a row's largest value in the sum: rows of one value 2^16 times the others, on a code of zero, were off by 2^-9.5 of the
// result, and rows of one sign, at groups of 128, by 5e-7 of it (rms; 5e-8 this way).  That costs 13 x 1536 -> 30522 7.0 -> 7.4 us, 1 x 7168 -> 16384 11.9 -> 12.5, fp32
// 13.6 -> 14.9.  fp32 parts below 2^-133, bf16's last place, are lost: rows below 2^-109 are off by up to 2^-131.
__device__ __forceinline__ bf16x8 codes_of(uint32_t q) {
  // (asm: what the compiler makes of the bytes otherwise are shifts of their own)
  uint32_t low = q ^ 0x88888888u, high;
  asm("" : "+v"(low));
  high = low >> 4;
  asm("" : "+v"(high));
  const auto value = [](uint32_t b) { return __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)b)); };
  const auto pair = [&](uint32_t even, uint32_t odd) { return __builtin_amdgcn_perm(value(odd), value(even), 0x07060302u); };
  return __builtin_bit_cast(bf16x8, u32x4{pair(low & 0xff, low >> 16 & 0xff), pair(high & 0xff, high >> 16 & 0xff), pair(low >> 8 & 0xff, low >> 24), pair(high >> 8 & 0xff, high >> 24)});
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
  // the values from the n-th on, 0 behind them
  __device__ __forceinline__ void drop(int n) {
    if (n & 4) v = u32x4{v[2], v[3], 0, 0};
    if (n & 2) v = u32x4{v[1], v[2], v[3], 0};
    if (n & 1) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    if (n >= 8) v = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ bf16x8 get(int) const { return __builtin_bit_cast(bf16x8, v); }
  __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  }
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
  __device__ __forceinline__ void drop(int n) {
    if (n & 4) v[0] = v[1], v[1] = u32x4{0, 0, 0, 0};
    if (n & 2) v[0] = u32x4{v[0][2], v[0][3], v[1][0], v[1][1]}, v[1] = u32x4{v[1][2], v[1][3], 0, 0};
    if (n & 1) v[0] = u32x4{v[0][1], v[0][2], v[0][3], v[1][0]}, v[1] = u32x4{v[1][1], v[1][2], v[1][3], 0};
    if (n >= 8) v[0] = v[1] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[i / 4][i % 4]);
  }
  __device__ __forceinline__ bf16x8 get(int lane) const {
    // part p is what x has in its first 8 (p + 1) bits and not in its first 8 p
    const int p = lane & 3;
    const uint32_t upto = p > 1 ? 0xffffffffu : p > 0 ? 0xffffff00u : 0xffff0000u, before = p > 1 ? 0xffffff00u : p > 0 ? 0xffff0000u : 0u;
    uint32_t f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = v[i / 4][i % 4];
      f[i] = __float_as_uint(__uint_as_float(x & upto) - __uint_as_float(x & before));
    }
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_perm(f[2 * i + 1], f[2 * i], 0x07060302u);      // the upper halves
    return __builtin_bit_cast(bf16x8, o);
  }
};

// The eight values of a row from column k on, 0 behind the last.  They are the last of the eight that end with the row, so that nothing is read one by one: that
// took 27.6 us for 16 x 1001 -> 30528, this way 9.3.  Rows of less than eight (SHORT) have no such eight.
template <typename T, bool SHORT>
__device__ __forceinline__ void load_edge(Operand<T>& to, const T* row, int k, int K) {
  if (SHORT) {
    to.one(row + k, K - k);
  } else {
    const int from = min(k, K - 8);
    to.load(row + from);
    to.drop(k - from);
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
template <typename T, int GROUP, bool SHORT, int NT>
struct Step {
  u32x4 q[NT];
  Scales<GROUP> s[NT];
  Operand<T> x[4];
  // `w`: the first tile's part, the others' `apart` bytes behind one another; those from `tiles` on are the last one again
  // and `EDGE`: whether this may be the end of a row
  template <bool EDGE>
  __device__ __forceinline__ void load(const unsigned char* w, long apart, int tiles, const T* row, int b, int K, int lane) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const unsigned char* p = w + min(t, tiles - 1) * apart + (long)b * tile_bytes(GROUP);
      q[t] = *reinterpret_cast<const u32x4*>(p + lane * 16);
      s[t].load(p, lane);
    }
    const int k = b * kTileK + (lane >> 4) * 8;
    if (!EDGE || (b + 1) * kTileK <= K) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i].load(row + k + i * 32);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) load_edge<T, SHORT>(x[i], row, k + i * 32, K);
    }
  }
  __device__ __forceinline__ void add(floatx4 (&sum)[NT], int lane) const {
    constexpr int kSteps = GROUP / 32;
#pragma unroll
    for (int g = 0; g < kTileK / GROUP; ++g) {
      bf16x8 a[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) a[i] = x[g * kSteps + i].get(lane);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        floatx4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) c = mfma(a[i], codes_of(q[t][g * kSteps + i]), c);
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

// Up to 16 rows of bf16 or 4 of fp32 (blockIdx.y of them).  A wave has NT tiles of 16 rows of W, and of their tiles of 128 columns every SPLIT-th; the SPLIT waves' sums meet in shared
// memory.
template <typename T, int GROUP, bool SHORT, int NT, int SPLIT>
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
    Step<T, GROUP, SHORT, NT> now, next;
    // from the last tile to the first, so that the end of a row is no matter of the loop
    if (part < kt) {
      int b = part + (kt - 1 - part) / SPLIT * SPLIT;
      now.template load<true>(mine, apart, tiles - t0, row, b, K, lane);
      for (; b >= 0; b -= SPLIT) {
        if (b >= SPLIT) next.template load<false>(mine, apart, tiles - t0, row, b - SPLIT, K, lane);
        now.add(sum, lane);
        now = next;
      }
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
      if (m < M) put(out, (long)m * N + n, fmaf(16.f, (sum[t][2] + sum[t][1]) + sum[t][0], b), gelu);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + (lane >> 4) * 4 + i;
        if (m < M) put(out, (long)m * N + n, fmaf(16.f, sum[t][i], b), gelu);
      }
    }
  }
}

// More rows: a workgroup has MT times 16 places of rows (as Operand) and 4 NT tiles of W's rows, NT a wave, SPLIT times (every SPLIT-th tile of 128
// columns, with sums that meet at the end).  x goes through shared memory, one tile of 128 columns after the other in two buffers, in the operand's order: 64 lanes times 16 bytes for each 16 places and 32 columns.  A lane's place among
// the 16 of its eighth is turned by the number of the eighth, so that the threads that write a row's sixteen eighths meet in no bank; readers are permuted
// among themselves.
template <typename T, bool SHORT, int MT>
struct Staged {
  static constexpr int kRows = MT * Operand<T>::kRows, kBytes = MT * 4 * 1024, kEach = kRows / 16;      // kEach: eighths of a thread
  static_assert(kRows % 16 == 0, "a row for every 16 threads");
  Operand<T> v[kEach];
  __device__ __forceinline__ void load(const T* x, long x_row, int m0, int M, int b, int K, int tid) {
    const int k = b * kTileK + (tid & 15) * 8;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const T* row = x + (long)min(m0 + (tid >> 4) + 16 * i, M - 1) * x_row;
      if ((b + 1) * kTileK <= K) v[i].load(row + k); else load_edge<T, SHORT>(v[i], row, k, K);
    }
  }
  __device__ __forceinline__ void store(unsigned char* to, int tid) const {
    const int c = tid & 15;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int row = (tid >> 4) + 16 * i;
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

template <typename T, int GROUP, bool SHORT, int MT, int NT, int SPLIT>
__global__ __launch_bounds__(256 * SPLIT, SPLIT > 2 ? SPLIT : 2) void int4_rows_kernel(const T* __restrict__ x, long x_row, const unsigned char* __restrict__ w, const float* __restrict__ bias,
                                                        T* __restrict__ out, int M, int N, int K, int gelu, int row_blocks) {
  constexpr int kSteps = GROUP / 32;
  __shared__ __attribute__((aligned(16))) unsigned char staged[SPLIT][2][Staged<T, SHORT, MT>::kBytes];
  const int tid = threadIdx.x & 255, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3, part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int tiles = (N + kTileN - 1) / kTileN, kt = (K + kTileK - 1) / kTileK;
  const int m0 = (int)(blockIdx.x % row_blocks) * Staged<T, SHORT, MT>::kRows, t0 = ((int)(blockIdx.x / row_blocks) * 4 + wave) * NT;
  const unsigned char* mine[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) mine[t] = w + (long)min(t0 + t, tiles - 1) * kt * tile_bytes(GROUP);
  floatx4 sum[MT][NT] = {};
  Staged<T, SHORT, MT> x_now;
  u32x4 q[NT], q_next[NT];
  Scales<GROUP> s[NT], s_next[NT];
  const auto ask = [&](int b) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const unsigned char* p = mine[t] + (long)b * tile_bytes(GROUP);
      q_next[t] = *reinterpret_cast<const u32x4*>(p + lane * 16);
      s_next[t].load(p, lane);
    }
    x_now.load(x, x_row, m0, M, b, K, tid);
  };
  if (part < kt) {
    ask(part);
    x_now.store(staged[part][0], tid);
  }
  __syncthreads();
  for (int n = 0, b = part; n * SPLIT < kt; ++n, b += SPLIT) {
    const bool more = b + SPLIT < kt;
    if (SPLIT > 1 && b >= kt) {      // other parts have a tile more
      __syncthreads();
      break;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) q[t] = q_next[t], s[t] = s_next[t];
    if (more) ask(b + SPLIT);
    const unsigned char* from = staged[part][n & 1];
#pragma unroll
    for (int g = 0; g < kTileK / GROUP; ++g) {
      bf16x8 a[MT][kSteps];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < kSteps; ++i) a[m][i] = Staged<T, SHORT, MT>::read(from, m, g * kSteps + i, lane);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bf16x8 v[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) v[i] = codes_of(q[t][g * kSteps + i]);
        const float scale = s[t].get(g);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          floatx4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kSteps; ++i) c = mfma(a[m][i], v[i], c);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[m][t][i] = fmaf(scale, c[i], sum[m][t][i]);
        }
      }
    }
    if (more) x_now.store(staged[part][(n + 1) & 1], tid);
    __syncthreads();
  }
  if (SPLIT > 1) {
    // the parts' sums meet where their rows were; each part takes a share of the tiles on
    static_assert(NT <= 2, "sums fit into a part's two stages");
    floatx4* const mine_sums = reinterpret_cast<floatx4*>(staged[part]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t) mine_sums[(m * NT + t) * 256 + tid] = sum[m][t];
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = (t0 + t) * kTileN + (lane & 15);
    if (n >= N) continue;
    const float bn = bias ? bias[n] : 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (SPLIT > 1) {
        if ((m * NT + t) % SPLIT != part) continue;
        sum[m][t] = reinterpret_cast<const floatx4*>(staged[0])[(m * NT + t) * 256 + tid];
#pragma unroll
        for (int p = 1; p < SPLIT; ++p) sum[m][t] += reinterpret_cast<const floatx4*>(staged[p])[(m * NT + t) * 256 + tid];
      }
      if constexpr (sizeof(T) == 4) {
        const int row = m0 + m * 4 + (lane >> 4);
        if (row < M) put(out, (long)row * N + n, fmaf(16.f, (sum[m][t][2] + sum[m][t][1]) + sum[m][t][0], bn), gelu);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = m0 + m * 16 + (lane >> 4) * 4 + i;
          if (row < M) put(out, (long)row * N + n, fmaf(16.f, sum[m][t][i], bn), gelu);
        }
      }
    }
  }
}

// Many rows.  Products of 16-bit floats are exact where x is: q - 8 has three bits and a scale eight, so (q - 8) s is a half-precision number of 11, and W needs
// no sums of its own for the scales.  What half precision lacks is range: rows of W come with a power of two that takes their largest scale below 2^11 (behind the
// tiles of `weight`, scale_factor), rows of x are taken to 2^14 .. 2^15 by one of their own, and the result is multiplied with both.  bf16 values below 2^-31 of their row's largest lose bits
// (2^-39 of that at most).  fp32 rows are two parts: x rounded to 11 bits, and 2^11 times what is left, with sums of its own, rounded to 11 bits too, so that a value is off by 2^-23 of itself at most, and
// those below 2^-27 of their row's largest by 2^-50 of that.  (With both in one sum, the second part lost bits from 2^-17 of the largest on: rows with one value 2^24 times the others, on a code of
// zero, were off by 2^-15.8 of the result, now 2^-22.)  Scales below 2^-27 of their row's largest lose bits (2^-36 of that at most).
//
// int4_operand_kernel writes x in that form once, in the order the matrix instructions take it in: 1024 bytes (Operand) for 16 rows, 32 columns and a part.
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// Four rows a workgroup, so that what it writes are pieces of 64 bytes.
template <typename T>
__global__ __launch_bounds__(256) void int4_operand_kernel(const T* __restrict__ x, long x_row, half8* __restrict__ out, int* __restrict__ exponent, int M, int K) {
  constexpr int kParts = sizeof(T) / 2, kHeld = 16 / kParts;      // kHeld: eighths that stay in registers between the two passes (rows of up to 8192, fp32 4096)
  __shared__ float most_of[4][4];
  const int tid = threadIdx.x, r = (int)blockIdx.x * 4 + (tid & 3), first = tid >> 2, kt = (K + kTileK - 1) / kTileK, end = r < M ? kt * 16 : 0;
  const T* row = x + (long)min(r, M - 1) * x_row;
  const auto load = [&](int c, Operand<T>& o) {      // eight columns, 0 behind the last
    if (c * 8 + 8 <= K) o.load(row + c * 8); else o.one(row + c * 8, K - c * 8);
  };
  float most = 0.f;
  const auto look = [&](const Operand<T>& o) {
    float v[8];
    o.values(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
  };
  Operand<T> held[kHeld];
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    if (first + h * 64 < end) load(first + h * 64, held[h]);
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    if (first + h * 64 < end) look(held[h]);
  for (int c = first + kHeld * 64; c < end; c += 64) {
    Operand<T> o;
    load(c, o);
    look(o);
  }
  for (int o = 32; o > 2; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
  if ((tid & 63) < 4) most_of[tid >> 6][tid & 3] = most;
  __syncthreads();
  most = fmaxf(fmaxf(most_of[0][tid & 3], most_of[1][tid & 3]), fmaxf(most_of[2][tid & 3], most_of[3][tid & 3]));
  // a row of zeros, or with an infinity, is taken as it is
  const int e = most > 0.f && most < __builtin_inff() ? 14 - ilogbf(most) : 0;
  if (tid < 4 && r < M) exponent[r] = -e;
  const auto write = [&](int c, const Operand<T>& o) {
    half8 part[kParts];
    float v[8];
    o.values(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = ldexpf(v[i], e);
      part[0][i] = (_Float16)f;
      if constexpr (kParts == 2) part[1][i] = (_Float16)((f - (float)part[0][i]) * 0x1p11f);
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p) out[((((long)(r / 16) * kt + c / 16) * kParts + p) * 4 + c / 4 % 4) * 64 + c % 4 * 16 + r % 16] = part[p];
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    if (first + h * 64 < end) write(first + h * 64, held[h]);
  for (int c = first + kHeld * 64; c < end; c += 64) {
    Operand<T> o;
    load(c, o);
    write(c, o);
  }
}

// (q & mask) | bits as one instruction, which takes one scalar register and no literals: the compiler is kept from knowing the two constants.
struct Codes {
  uint32_t mask, bits;
  __device__ __forceinline__ Codes(uint32_t m, uint32_t b) : mask(m), bits(b) { asm volatile("" : "+s"(mask), "+v"(bits)); }
  __device__ __forceinline__ uint32_t operator()(uint32_t q) const { return (q & mask) | bits; }
};

// Eight codes times a scale as (16 + q) s - 24 s, exactly: 0x4c00 is 16 and its bits from the seventh are worth 1, and 24 s has ten bits.
struct ScaledCodes : Codes {
  __device__ __forceinline__ ScaledCodes() : Codes(0x03c003c0u, 0x4c004c00u) {}
  __device__ __forceinline__ half8 get(uint32_t q, half2v s, half2v off) const {
    const Codes& c = *this;
    const auto pair = [&](uint32_t b) { return __builtin_elementwise_fma(__builtin_bit_cast(half2v, c(b)), s, off); };
    const half2v v[4] = {pair(q << 6), pair(q << 2), pair(q >> 2), pair(q >> 6)};
    return __builtin_bit_cast(half8, v);
  }
};
__device__ __forceinline__ floatx4 mfma(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// What a row's scales are multiplied with: its factor takes the largest to [1 / 2, 1), 2^11 more to [2^10, 2^11), as high as 24 times a scale goes, so that those 2^-27 of it are exact too.
// (The factor ends at 2^-120, where scales may be 2^8 yet, and 2^120.)
__device__ __forceinline__ float scale_factor(float f) { return f > 0x1p-120f ? fminf(f, 0x1p116f) * 0x1p11f : f * 4.f; }

// A workgroup has MT times 16 rows of x and WAVES NT tiles of W's rows, NT a wave, SPLIT times: every SPLIT-th tile of 128 columns, with sums that meet at
// the end.  x comes straight into shared memory, a tile of 128 columns ahead; W is made in registers, once for MT products.
template <typename T, int GROUP, int MT, int NT, int SPLIT, int WAVES>
__global__ __launch_bounds__(64 * WAVES * SPLIT, WAVES * SPLIT > 8 ? WAVES * SPLIT / 4 : 2) void int4_many_rows_kernel(const unsigned char* __restrict__ x, const int* __restrict__ exponent, const unsigned char* __restrict__ w,
                                                                const float* __restrict__ bias, T* __restrict__ out, int M, int N, int K, int gelu, int row_blocks, int col_blocks) {
  constexpr int kParts = sizeof(T) / 2, kStage = MT * kParts * 4096, kSteps = GROUP / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char staged[];      // two stages a part
  __shared__ int exponents[MT * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WAVES, part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / WAVES;
  const int tiles = (N + kTileN - 1) / kTileN, kt = (K + kTileK - 1) / kTileK, row_tiles = (M + 15) / 16;
  // workgroups of the same columns behind one another on the same XCD (they are dealt to the eight in turn)
  const int at = (int)blockIdx.x / 8, col = at / row_blocks * 8 + (int)blockIdx.x % 8;
  if (col >= col_blocks) return;
  const int m0 = at % row_blocks * MT, t0 = (col * WAVES + wave) * NT;
  const unsigned char* mine[NT];
  float row_factor[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int tile = min(t0 + t, tiles - 1);
    mine[t] = w + (long)tile * kt * tile_bytes(GROUP);
    row_factor[t] = scale_factor(reinterpret_cast<const float*>(w + (long)tiles * kt * tile_bytes(GROUP))[tile * 16 + (lane & 15)]);
  }
  // what the end needs is asked for now
  if (threadIdx.x < MT * 16) exponents[threadIdx.x] = exponent[min(m0 * 16 + (int)threadIdx.x, M - 1)];
  const int n0 = t0 * kTileN;
  float bn[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) bn[t] = bias && n0 + t * 16 + (lane & 15) < N ? bias[n0 + t * 16 + (lane & 15)] : 0.f;
  floatx4 sum[kParts][MT][NT] = {};
  u32x4 q[NT], q_next[NT];
  Scales<GROUP> s[NT], s_next[NT];
  half2v scale[NT], off[NT];
  const ScaledCodes codes;
  const unsigned lds0 = (unsigned)(uintptr_t)staged + part * 2 * kStage;
  const auto ask = [&](int b, int stage) {
    // pieces of 1024 bytes, dealt to the waves
#pragma unroll
    for (int i = 0; i < MT * kParts * 4 / WAVES; ++i) {
      const int piece = i * WAVES + wave, m = piece / (4 * kParts);
      const unsigned char* from = x + (((long)min(m0 + m, row_tiles - 1) * kt + b) * kParts * 4 + piece % (4 * kParts)) * 1024;
      load_to_lds(lds0 + stage * kStage + piece * 1024, lane * 16, from);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const unsigned char* p = mine[t] + (long)b * tile_bytes(GROUP);
      q_next[t] = *reinterpret_cast<const u32x4*>(p + lane * 16);
      s_next[t].load(p, lane);
    }
  };
  if (part < kt) ask(part, 0);
  for (int n = 0, b = part; n * SPLIT < kt; ++n, b += SPLIT) {
#pragma unroll
    for (int t = 0; t < NT; ++t) q[t] = q_next[t], s[t] = s_next[t];
    __builtin_amdgcn_s_waitcnt(kWaitVm0);      // this tile of x is there, of this wave's pieces
    __syncthreads();                           // of all; and nobody reads the other stage any more
    if (SPLIT > 1 && b >= kt) break;           // other parts have a tile more
    if (b + SPLIT < kt) ask(b + SPLIT, (n + 1) & 1);
    const unsigned char* from = staged + (part * 2 + (n & 1)) * kStage + lane * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      half8 a[kParts][MT];
#pragma unroll
      for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int m = 0; m < MT; ++m) a[p][m] = *reinterpret_cast<const half8*>(from + ((m * kParts + p) * 4 + i) * 1024);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (i % kSteps == 0) {
          const _Float16 one = (_Float16)(s[t].get(i / kSteps) * row_factor[t]);
          scale[t] = half2v{one, one};
          off[t] = scale[t] * half2v{(_Float16)-24.f, (_Float16)-24.f};
        }
        const half8 v = codes.get(q[t][i], scale[t], off[t]);
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
          for (int m = 0; m < MT; ++m) sum[p][m][t] = mfma(a[p][m], v, sum[p][m][t]);
      }
    }
  }
  // the parts of x together: the second is 2^11 times what it stands for
  if constexpr (kParts == 2)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[0][m][t][i] = fmaf(sum[1][m][t][i], 0x1p-11f, sum[0][m][t][i]);
  // 16 rows at a time through shared memory, each wave by itself, so that a row's values leave together
  constexpr int kRow = NT * 16 + 4;
  __syncthreads();
  if (SPLIT > 1) {      // the parts' sums meet where their rows were
    static_assert(SPLIT == 1 || NT * WAVES <= 8 * kParts, "sums fit into a part's two stages");
    floatx4* const sums = reinterpret_cast<floatx4*>(staged + part * 2 * kStage) + threadIdx.x % (64 * WAVES);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t) sums[(m * NT + t) * 64 * WAVES] = sum[0][m][t];
    __syncthreads();
  }
  float* const mine_out = reinterpret_cast<float*>(staged + (SPLIT > 1 ? SPLIT * 2 * kStage : 0)) + (threadIdx.x >> 6) * 16 * kRow;
  // the powers of two are put together as exponents: as numbers their product may be out of range where the result is not
  int en[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) en[t] = 127 - (int)(__float_as_uint(row_factor[t]) >> 23);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if ((m0 + m) * 16 >= M) break;
    if (SPLIT > 1) {
      if (m % SPLIT != part) continue;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const floatx4* sums = reinterpret_cast<const floatx4*>(staged) + (m * NT + t) * 64 * WAVES + threadIdx.x % (64 * WAVES);
        sum[0][m][t] = sums[0];
#pragma unroll
        for (int p = 1; p < SPLIT; ++p) sum[0][m][t] += sums[p * 2 * kStage / 16];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (lane >> 4) * 4 + i;
      const int em = exponents[m * 16 + row];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float y = ldexpf(sum[0][m][t][i], em + en[t]) + bn[t];
        if (gelu) y = gelu_erf(y);
        mine_out[row * kRow + t * 16 + (lane & 15)] = y;
      }
    }
    __builtin_amdgcn_wave_barrier();
    constexpr int kEach = NT * 4;      // values of a lane: a quarter of a row
    const int row = lane >> 2, at_n = (lane & 3) * kEach, R = (m0 + m) * 16 + row;
    float y[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i += 4) *reinterpret_cast<floatx4*>(y + i) = *reinterpret_cast<const floatx4*>(mine_out + row * kRow + at_n + i);
    __builtin_amdgcn_wave_barrier();
    if (R < M) {
      T* to = out + (long)R * N + n0 + at_n;
      const int left = N - n0 - at_n;
      if (left >= kEach) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < kEach; i += 4)
            *reinterpret_cast<u32x4_any*>(to + i) = u32x4_any{__float_as_uint(y[i]), __float_as_uint(y[i + 1]), __float_as_uint(y[i + 2]), __float_as_uint(y[i + 3])};
        } else if constexpr (kEach >= 8) {
#pragma unroll
          for (int i = 0; i < kEach; i += 8)
            *reinterpret_cast<u32x4_any*>(to + i) = u32x4_any{pack_bf16x2(y[i], y[i + 1]), pack_bf16x2(y[i + 2], y[i + 3]), pack_bf16x2(y[i + 4], y[i + 5]), pack_bf16x2(y[i + 6], y[i + 7])};
        } else {
          *reinterpret_cast<u32x2_any*>(to) = u32x2_any{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        }
      } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (i < left) put(to, i, y[i], 0);
      }
    }
  }
}

}  // namespace m2

using namespace m2;

extern "C" size_t m2_int4_weight_bytes(int N, int K, int group) {
  if (N <= 0 || K <= 0 || (group != 32 && group != 64 && group != 128)) return 0;
  const size_t tiles = (size_t)((N + kTileN - 1L) / kTileN);
  return tiles * ((size_t)((K + kTileK - 1L) / kTileK) * (size_t)tile_bytes(group) + kTileN * sizeof(float));
}

// Which kernel a product runs on, with how many times 16 places of rows (MT) and tiles of 16 rows of W (NT) a wave, and how many parts of K.
//
// What a wave takes for a tile of 128 columns is mostly waiting, so the smallest workgroups of one round over the chip win, and K is split as far as registers and
// shared memory go.  us, rows 2 1 1 (32 rows of bf16 or 16 of fp32 a workgroup, K whole) / the few rows' kernel over MT = 1, NT = 1 / 2 / 4 / rows 2 1 4 / many 4 1 4 / many 4 2 2, bf16, K -> N:
//   1792 -> 1792 M = 32 10.5 / 5.2 / 5.6 / 6.8 / 7.5; M = 128 10.6 / 10.2 / 7.5 / 6.9 / 7.7 / 13.4; M = 256 11.1 / 15.9 / 11.9 / 9.6 / 8.4 / 14.1
//   4096 -> 2000 M = 64 19.8 / 11.7 / 8.7 / 9.9 / 12.5 / 18.8; M = 256 22.9 / 35 / 23 / 16.3 / 13.6 / 21.1; M = 512 24.3 / - / - / - / 25.2 / 24.3
//   7168 -> 1792 M = 128 34.3 / 30.4 / 19.0 / 15.5 / 19.3 / 28.1; M = 512 38.3 / - / - / - / 39.2 / 32.7 / 43
//   4096 -> 8192 M = 64 23 / 34 / 21.5 / 16.4 / 13.9 / 19.6; M = 128 23.8 / 69 / 38 / 28 / 25 / 21.7 / 27.3; M = 256 38.5 / - / - / 49 / 47 / 36 / 30.0
// fp32 (rows 4 1 2 / many 1 1 4 / 2 1 4 / 2 2 2):
//   5672 -> 1200 M = 8 31 / 8.2 / 9.8 / 13.5 / 26.1; M = 64 32 / 27 / 21.4 / 28 / 26.2 / 23.3 / 26.8; M = 256 40 / - / - / 66 / 39 / 39 / 30.8 / 40
//   4096 -> 8192 M = 32 23.9 / 52 / 35 / 36 / 20.2 / 18.7 / 20.8; M = 64 31 / - / - / - / 31 / 28.6 / 23.0 / 28.9; M = 128 54 / - / - / - / 58 / 48 / 37.0 / 32.5
// many 2 2 1 / 2 2 2 / 3 2 2 / 4 2 2, groups of 32: 768 -> 30522 M = 40 16.0 / 18.8 / 14.3 / 15.6, M = 48 16.1 / 19.0 / 14.5 / 15.9, M = 64 16.8 / 19.6 / 22.1 / 16.9, 1536 -> 16000 M = 96
// 23.3 / 26.7 / 20.2 / 22.7, M = 128 25.1 / 27.9 / 31.0 / 23.6.
// Where x is written as half-precision operands first (kMany), that takes 4 us and more, which only a large product wins back.  us, rows / many: 768 -> 30528 bf16 M = 64 11.1 /
// 12.2, 128 17.9 / 16.1, 256 29.5 / 23.5; fp32 1792 -> 1792 M = 64 10.4 / 11.7, 768 -> 30522 M = 16 9.6 / 11.9, 40 19.9 / 14.3, 128 43 / 24.7.
// Its workgroups have 4 NT tiles, and 8 NT where as much of the chip is used: 768 -> 30528 M = 256 24.0 / 23.5, 1792 -> 16000 M = 512 41.5 / 40.8, 7168 -> 30528 M = 150 100 / 112 (717 and 360
// workgroups); fp32, 32 rows by 4 NT / 64 by 8 NT: 4096 -> 8192 M = 256 50.6 / 61.7, 512 85.7 / 73.4, 7168 -> 16384 M = 512 258 / 224.
// fp32 of 64 rows by 8 NT takes 144 registers with its two sums, so that one workgroup has a compute unit; 48 rows 120, which two share: 512 rows, 64 / 48: 768 -> 30528 68.0 / 61.9 (960 and 1320
// workgroups), 7168 -> 16384 224 / 235 (512, 704), 4096 -> 8192 73.4 / 87.4 (256, 352).
struct Plan {
  enum Kernel { kFew, kRows, kMany } kernel;
  int mt, nt, split, waves = 4;      // waves: of kMany, times split
};
static Plan plan_of(int M, int N, int K, int dtype) {
  const bool f32 = dtype == M2_DTYPE_F32;
  const long tiles = (N + kTileN - 1L) / kTileN, kt = (K + kTileK - 1L) / kTileK, round = num_cus();
  const long places = f32 ? (M + 3L) / 4 : (M + 15L) / 16;      // times 16 places of an operand
  const auto blocks = [&](int rows, int columns) { return (M + rows - 1L) / rows * ((tiles + columns - 1) / columns); };      // of `rows` rows and `columns` tiles
  if (places == 1) {
    // Few tiles: all of a workgroup's waves share one.  More: tiles share what a wave reads (and splits) of x, four where that is as much as a tile, and
    // long rows are shared by eight waves, short ones by four where there are many tiles and a wave has little more to do.  us, NT and SPLIT 1, 8 / 2, 4 / 2, 8 / 4, 4 / 4, 8: 768 -> 768 M = 1 3.5 / 3.9 / 3.7 / 4.6 / 4.3;
    // 4096 -> 4096 M = 16 7.6 / 9.3 / 8.1 / 12.1 / 10.4; 1792 -> 7168 M = 16 6.9 / 6.3 / 5.8 / 7.6 / 6.9; 768 -> 30528 M = 1 5.9 / 5.7 / 6.3 / 6.6 / 5.9, M = 16 9.4 / 7.4 / 8.0 / 7.7 / 6.8; 1536 ->
    // 30522 M = 16 15.6 / 11.1 / 11.5 / 10.0 / 9.3, M = 9 11.4 / 9.6 / 9.7 / 9.5 / 8.8; 4096 -> 16384 M = 1 10.2 / 11.2 / 10.3 / 12.8 / 11.1, M = 16 19.6 / 13.1 / 13.3 / 13.7 / 11.9; 1792 -> 15000
    // M = 1 6.7 / 7.5 / 6.7 / 8.8 / 7.2; fp32 768 -> 17000 M = 1 6.4 / 5.6 / 5.6 / 6.8 / 7.0, 768 -> 30522 M = 4 9.3 / 6.6 / 7.4 / 7.3 / 7.8, 1536 -> 30522 M = 4 13.1 / 10.5 / 10.2 / 9.8 / 11.1, 7168 ->
    // 16384 M = 1 25.3 / 22.0 / 19.0 / 22.7 / 18.2.
    if (K < 8 || tiles < 384) return {Plan::kFew, 1, 1, 8};
    const bool many = tiles >= 1536 || (kt >= 16 && tiles >= 1024);
    if (!many) return {Plan::kFew, 1, 2, 8};
    if (f32) return {Plan::kFew, 1, kt < 8 ? 2 : 4, kt < 16 ? 4 : 8};
    return M > 8 ? Plan{Plan::kFew, 1, 4, 8} : Plan{Plan::kFew, 1, 2, kt < 16 ? 4 : 8};
  }
  if (K >= 8)
    for (int nt = 1; nt <= 4; nt *= 2)
      if (places * ((tiles + nt - 1) / nt) <= round) return {Plan::kFew, 1, nt, 8};
  const double products = (double)M * N * K;
  if (f32) {
    if (products >= 4e8) {
      if (blocks(16, 4) <= round) return {Plan::kMany, 1, 1, 4};
      if (blocks(32, 4) <= round) return {Plan::kMany, 2, 1, 4};
      for (int mt = 2; mt <= 4; ++mt)
        if (blocks(16 * mt, 8) <= round) return {Plan::kMany, mt, 2, 2};
      if (blocks(64, 16) >= round) return {Plan::kMany, blocks(64, 16) > 2 * round ? 3 : 4, 2, 1, 8};
      return {Plan::kMany, 2, 2, 1};
    }
    if (K >= 8 && blocks(16, 4) <= round) return {Plan::kRows, 4, 1, 2};
    return {Plan::kRows, 4, K >= 8 && blocks(16, 8) >= 2 * round ? 2 : 1, 1};
  }
  if (K >= 8 && blocks(32, 4) <= round) return {Plan::kRows, 2, 1, 4};
  if (M > 64 && products >= 3e9) {
    if (blocks(64, 4) <= round) return {Plan::kMany, 4, 1, 4};
    if (blocks(64, 8) <= round) return {Plan::kMany, 4, 2, 2};
    // what of its last round over the chip is in use
    const auto use = [&](long b) { return (double)b / (double)((b + round - 1) / round * round); };
    return {Plan::kMany, 4, 2, 1, use(blocks(64, 16)) > 0.9 * use(blocks(64, 8)) ? 8 : 4};
  }
  if (K >= 8 && blocks(32, 4) <= 2 * round) return {Plan::kRows, 2, 1, 2};
  return {Plan::kRows, 2, K >= 8 && blocks(32, 8) >= 2 * round ? 2 : 1, 1};
}

extern "C" size_t m2_int4_workspace_bytes(int M, int N, int K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || plan_of(M, N, K, dtype).kernel != Plan::kMany) return 0;
  const size_t row_tiles = (size_t)((M + 15L) / 16), kt = (size_t)((K + kTileK - 1L) / kTileK);
  return row_tiles * (kt * (dtype == M2_DTYPE_F32 ? 8192 : 4096) + 16 * sizeof(int));
}

extern "C" int m2_int4_linear_fwd(const void* x, long x_row, const void* weight, const float* bias, void* out, void* workspace, int M, int N, int K, int group, int gelu,
                                  int dtype, void* stream) {
  const char* who = "m2_int4_linear_fwd";
  if (!x || !weight || !out) return set_error(M2_ERR_ARG, "%s: null pointer", who);
  if (dtype != M2_DTYPE_F32 && dtype != M2_DTYPE_BF16) return set_error(M2_ERR_ARG, "%s: dtype must be M2_DTYPE_F32 or M2_DTYPE_BF16 (got %d)", who, dtype);
  if (M <= 0 || N <= 0 || K <= 0 || x_row < 0 || (gelu != 0 && gelu != 1)) return set_error(M2_ERR_ARG, "%s: M=%d N=%d K=%d x_row=%ld gelu=%d", who, M, N, K, x_row, gelu);
  if (N > kMaxSize || K > kMaxSize) return set_error(M2_ERR_UNSUPPORTED, "%s: N and K of at most 2^30 (N=%d K=%d)", who, N, K);
  if (group != 32 && group != 64 && group != 128) return set_error(M2_ERR_UNSUPPORTED, "%s: groups of 32, 64 or 128 values (got %d)", who, group);
  if (!aligned16(weight, workspace)) return set_error(M2_ERR_UNSUPPORTED, "%s: weight and workspace must be 16-byte aligned", who);
  if (!workspace && m2_int4_workspace_bytes(M, N, K, dtype)) return set_error(M2_ERR_ARG, "%s: M=%d rows need a workspace", who, M);
  const uintptr_t size = dtype == M2_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)x % size || (uintptr_t)out % size || (uintptr_t)bias % 4) return set_error(M2_ERR_UNSUPPORTED, "%s: x, out and bias must be aligned to their type", who);
  hipStream_t st = (hipStream_t)stream;
  const int tiles = (int)((N + kTileN - 1L) / kTileN), kt = (int)((K + kTileK - 1L) / kTileK);
  // a launch holds below 2^32 threads
  const auto fits = [](long blocks, long threads) { return blocks < (1L << 32) / threads; };
  const auto too_large = [&] { return set_error(M2_ERR_UNSUPPORTED, "%s: M=%d N=%d K=%d are more workgroups than a launch holds", who, M, N, K); };
  const auto go = [&](auto kernel, auto* t, int nt, int split) {
    using T = std::remove_pointer_t<decltype(t)>;
    const long waves = (tiles + nt - 1L) / nt * split, each = waves_of(split), blocks = (waves + each - 1) / each, places = (M + Operand<T>::kRows - 1L) / Operand<T>::kRows;
    if (!fits(blocks * places, 64 * each)) return too_large();
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)places), dim3(64 * each), 0, st, (const T*)x, x_row, (const unsigned char*)weight, bias, (T*)out, M, N, K, gelu);
    return check_launch("int4_linear");
  };
  const auto many = [&](auto kernel, auto* t, int mt, int nt, int split, int waves) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int row_tiles = (int)((M + 15L) / 16), row_blocks = (row_tiles + mt - 1) / mt, col_blocks = (tiles + waves * nt - 1) / (waves * nt), parts = (int)sizeof(T) / 2;
    const long blocks = (col_blocks + 7L) / 8 * 8 * row_blocks;
    if (!fits(blocks, 64 * waves * split) || !fits((M + 3L) / 4, 256)) return too_large();
    int* exponent = (int*)((unsigned char*)workspace + (size_t)row_tiles * kt * parts * 4096);
    const int stages = split * 2 * mt * parts * 4096, leave = split * waves * 16 * (nt * 16 + 4) * 4, lds = split > 1 ? stages + leave : stages > leave ? stages : leave;
    if (lds > 64 * 1024) {
      const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return set_error(M2_ERR_LAUNCH, "hipFuncSetAttribute(int4_many_rows): %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL((int4_operand_kernel<T>), dim3((unsigned)((M + 3) / 4)), dim3(256), 0, st, (const T*)x, x_row, (half8*)workspace, exponent, M, K);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * waves * split), (size_t)lds, st, (const unsigned char*)workspace, exponent,
                       (const unsigned char*)weight, bias, (T*)out, M, N, K, gelu, row_blocks, col_blocks);
    return check_launch("int4_linear");
  };
  const auto rows = [&](auto kernel, auto* t, int mt, int nt, int split) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int each = mt * Operand<T>::kRows, row_blocks = (int)((M + each - 1L) / each);
    const long blocks = (tiles + 4L * nt - 1) / (4 * nt) * row_blocks;
    if (!fits(blocks, 256 * split)) return too_large();
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256 * split), 0, st, (const T*)x, x_row, (const unsigned char*)weight, bias,
                       (T*)out, M, N, K, gelu, row_blocks);
    return check_launch("int4_linear");
  };
  const Plan p = plan_of(M, N, K, dtype);
  const auto parts = [&](auto* t, auto g) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int G = decltype(g)::value;
    constexpr bool kF32 = sizeof(T) == 4;
    if (p.kernel == Plan::kFew) {
      if (K < 8) return go(int4_few_rows_kernel<T, G, true, 1, 8>, t, 1, 8);
      if (p.nt == 1) return go(int4_few_rows_kernel<T, G, false, 1, 8>, t, 1, 8);
      if (p.nt == 2) return p.split == 4 ? go(int4_few_rows_kernel<T, G, false, 2, 4>, t, 2, 4) : go(int4_few_rows_kernel<T, G, false, 2, 8>, t, 2, 8);
      if constexpr (kF32)
        if (p.split == 4) return go(int4_few_rows_kernel<T, G, false, 4, 4>, t, 4, 4);
      return go(int4_few_rows_kernel<T, G, false, 4, 8>, t, 4, 8);
    }
    if (p.kernel == Plan::kRows) {
      constexpr int kMt = kF32 ? 4 : 2;
      if (K < 8) return rows(int4_rows_kernel<T, G, true, kMt, 1, 1>, t, kMt, 1, 1);
      if (p.nt == 2) return rows(int4_rows_kernel<T, G, false, kMt, 2, 1>, t, kMt, 2, 1);
      if (p.split == 1) return rows(int4_rows_kernel<T, G, false, kMt, 1, 1>, t, kMt, 1, 1);
      if (kF32 || p.split == 2) return rows(int4_rows_kernel<T, G, false, kMt, 1, 2>, t, kMt, 1, 2);
      if constexpr (!kF32) return rows(int4_rows_kernel<T, G, false, kMt, 1, 4>, t, kMt, 1, 4);
    }
    constexpr int kMt = kF32 ? 2 : 4;
    if (p.nt == 2 && p.split == 2) {
      if (p.mt == 4) return many(int4_many_rows_kernel<T, G, 4, 2, 2, 4>, t, 4, 2, 2, 4);
      if constexpr (kF32) return p.mt == 3 ? many(int4_many_rows_kernel<T, G, 3, 2, 2, 4>, t, 3, 2, 2, 4) : many(int4_many_rows_kernel<T, G, 2, 2, 2, 4>, t, 2, 2, 2, 4);
    }
    if constexpr (kF32)
      if (p.nt == 2 && p.waves == 8 && p.mt == 3) return many(int4_many_rows_kernel<T, G, 3, 2, 1, 8>, t, 3, 2, 1, 8);
    if (p.nt == 2 && p.waves == 8) return many(int4_many_rows_kernel<T, G, 4, 2, 1, 8>, t, 4, 2, 1, 8);
    if constexpr (kF32) {
      if (p.nt == 2) return many(int4_many_rows_kernel<T, G, 2, 2, 1, 4>, t, 2, 2, 1, 4);
      if (p.mt == 1) return many(int4_many_rows_kernel<T, G, 1, 1, 4, 4>, t, 1, 1, 4, 4);
    }
    if constexpr (!kF32)
      if (p.nt == 2) return many(int4_many_rows_kernel<T, G, 4, 2, 1, 4>, t, 4, 2, 1, 4);
    return many(int4_many_rows_kernel<T, G, kMt, 1, 4, 4>, t, kMt, 1, 4, 4);
  };
  const auto pick = [&](auto* t) {
    if (group == 32) return parts(t, std::integral_constant<int, 32>{});
    if (group == 64) return parts(t, std::integral_constant<int, 64>{});
    return parts(t, std::integral_constant<int, 128>{});
  };
  return dtype == M2_DTYPE_F32 ? pick((float*)nullptr) : pick((uint16_t*)nullptr);
}
