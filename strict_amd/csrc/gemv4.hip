// Products of a few rows of 16-bit activations with a matrix of 4-bit weights
// (sh_gemv_w4a16_*), and the weights' quantisation and layout.
//
// y[b][n] = sum over groups g of 32 columns of 2^(scale[n][g] - 127) sum_k x[b][k] w[n][k],
// w one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (OCP E2M1, MX scales).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "common.h"
#include "gemv4.h"
#include "paged.h"
#include "paged_device.h"

namespace sh {
namespace {

constexpr int kT = 256;

// ---- quantisation and layout ---------------------------------------------------------

// A thread a group: the smallest scale 2^e, e >= -127, for which its largest value is at
// most 6 * 2^e = 1.5 * 2^(e + 2), each value to the nearest (half way: the even one). Bound
// by the bytes: 151,936 x 1,024 125 us (705 MB, 5.6 TB/s).
__global__ __launch_bounds__(kT) void quantize_e2m1_kernel(const float *__restrict__ W, size_t groups, uint8_t *q,
                                                           uint8_t *scales) {
  const size_t g = (size_t)blockIdx.x * kT + threadIdx.x;
  if (g >= groups) return;
  float w[32];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(W + g * 32 + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; e++) w[4 * i + e] = v[e];
  }
  float most = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 32; i++) {
    finite = finite && __builtin_fabsf(w[i]) < INFINITY;
    most = fmaxf(most, __builtin_fabsf(w[i]));
  }
  const uint32_t bits = __builtin_bit_cast(uint32_t, most);
  const int e = max((int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffff) > 0x400000 ? 1 : 0), -127);
  const float to_group = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);  // 2^-e, e of -127 .. 126
  u32x4 code;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, w[8 * i] * to_group, w[8 * i + 1] * to_group, 1.0f, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, w[8 * i + 2] * to_group, w[8 * i + 3] * to_group, 1.0f, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, w[8 * i + 4] * to_group, w[8 * i + 5] * to_group, 1.0f, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, w[8 * i + 6] * to_group, w[8 * i + 7] * to_group, 1.0f, 3);
    code[i] = d;
  }
  *reinterpret_cast<u32x4 *>(q + g * 16) = finite ? code : u32x4{0, 0, 0, 0};
  scales[g] = finite ? (uint8_t)(e + 127) : 255;
}

// Scales 2^e with which every weight but 0 (0.5 to 6 times it) is a normal number.
constexpr int kF16Least = 127 - 13, kF16Most = 127 + 13, kBf16Least = 127 - 125, kBf16Most = 127 + 125;

constexpr int kPackT = 1024;

// A workgroup takes 16 rows, its waves their tiles in turn. A group of zeros gets the scale 1,
// whatever its own. (12,289 x 8,160 34 us, 4,096 x 4,096 11; a wave for 16 rows 122 and 36.)
__global__ __launch_bounds__(kPackT) void pack_e2m1_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ scales,
                                                       int N, int K, int col_tiles, uint8_t *w, uint32_t *tile_scales,
                                                       uint32_t *tile_flags) {
  __shared__ uint32_t row_flags;
  const int lane = threadIdx.x & 63, r16 = lane & 15, grp = lane >> 4, waves = blockDim.x >> 6;
  const size_t tile = blockIdx.x, row = tile * 16 + r16;
  if (threadIdx.x == 0) row_flags = 0;
  __syncthreads();
  const bool there = row < (size_t)N;
  bool nan = false, no_f16 = false, no_bf16 = false;
  for (size_t t = threadIdx.x >> 6; t < (size_t)col_tiles; t += waves) {
    u32x4 code = {0, 0, 0, 0};
    uint32_t scale = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const size_t group = t * 4 + j;
      uint32_t s = 127;
      bool some = false;
      if (there && group * 32 < (size_t)K) {
        code[j] = *reinterpret_cast<const uint32_t *>(q + row * (K / 2) + group * 16 + grp * 4);
        s = scales[row * (K / 32) + group];
        some = (code[j] & 0x77777777u) != 0;
      }
      int row_some = some ? 1 : 0;
      row_some |= __shfl_xor(row_some, 16, 64);
      row_some |= __shfl_xor(row_some, 32, 64);
      some = row_some != 0;
      if (s == 255)
        nan = true;
      else if (some) {
        no_f16 = no_f16 || s < kF16Least || s > kF16Most;
        no_bf16 = no_bf16 || s < kBf16Least || s > kBf16Most;
      }
      scale |= (some && s != 255 ? s : 127u) << (8 * j);
    }
    *reinterpret_cast<u32x4 *>(w + (tile * col_tiles + t) * 1024 + lane * 16) = code;
    if (grp == 0) tile_scales[(tile * col_tiles + t) * 16 + r16] = scale;
  }
  const uint32_t nans = (uint32_t)__ballot(nan) & 0xffffu;
  const uint32_t flags = nans | (__any(no_f16) ? 1u << 16 : 0) | (__any(no_bf16) ? 1u << 17 : 0);
  if (lane == 0 && flags != 0) atomicOr(&row_flags, flags);
  __syncthreads();
  if (threadIdx.x == 0) tile_flags[tile] = row_flags;
}

// ---- the products ----------------------------------------------------------------------

struct Gemv4Args {
  const uint16_t *x;
  const uint8_t *w, *scales;
  const uint32_t *flags;
  void *y;
  int batch, K, N, ldx, row_tiles, col_tiles;
  size_t ldy;
};

// Eight weights of a dword times the power of two in `scale`, in the 16-bit type.
template <class T>
__device__ __forceinline__ typename T::Vec from_e2m1(uint32_t eight, float scale) {
  u32x4 v;
  if constexpr (T::kIsF16)
    v = u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 0)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 2)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 3))};
  else
    v = u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(eight, scale, 0)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(eight, scale, 1)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(eight, scale, 2)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(eight, scale, 3))};
  return __builtin_bit_cast(typename T::Vec, v);
}

// The nearest exponent with which every weight is a normal number of the type.
template <class T>
__device__ __forceinline__ uint32_t normal_exponent(uint32_t exponent) {
  constexpr uint32_t kLeast = T::kIsF16 ? kF16Least : kBf16Least, kMost = T::kIsF16 ? kF16Most : kBf16Most;
  return min(max(exponent, kLeast << 23), kMost << 23);
}

// What a wave has of a step: kR tiles of weights, their scales, and the activations.
template <int kR>
struct Gemv4Step {
  u32x4 w[kR], x[4];
  uint32_t s[kR];
};

// Up to 16 rows of activations. A workgroup takes kR tiles of rows; its waves share the
// columns, step by step of 128 in turn, and add up in LDS in their order. Activations are
// the rows of the products, weights the columns, so that a lane's results are of one row of
// weights; row b of x is the product's row 4 (b % 4) + b / 4, so that up to 4 of them need
// one register (kI) and up to 8 two. Where a scale leaves the type's normal numbers
// (kExact), weights are converted with the nearest that does not, and each group's sum is
// multiplied by the rest. Bound by the weights' bytes.
template <class T, int kR, int kI, bool kExact>
__device__ __forceinline__ void gemv4_sum(const Gemv4Args &a, f32x4 (&acc)[kR]) {
  typedef typename T::Vec Vec;
  const int lane = threadIdx.x & 63, r16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const uint16_t *x = a.x + (size_t)min(4 * (r16 & 3) + (r16 >> 2), a.batch - 1) * a.ldx + grp * 8;
  size_t first[kR];
#pragma unroll
  for (int r = 0; r < kR; r++) first[r] = (size_t)min((int)blockIdx.x * kR + r, a.row_tiles - 1) * a.col_tiles;
  auto load = [&](int t, Gemv4Step<kR> &s) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < kR; r++) {
      s.w[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(a.w + (first[r] + t) * 1024 + lane * 16));
      s.s[r] = *reinterpret_cast<const uint32_t *>(a.scales + (first[r] + t) * 64 + r16 * 4);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) s.x[j] = *reinterpret_cast<const u32x4 *>(x + min(128 * t + 32 * j, a.K - 32));
  };
  auto multiply = [&](int t, Gemv4Step<kR> &s) __attribute__((always_inline)) {
    if (128 * t + 128 > a.K) {  // columns behind the last: zeros, whatever x has there
#pragma unroll
      for (int j = 1; j < 4; j++)
        if (128 * t + 32 * j >= a.K) s.x[j] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int r = 0; r < kR; r++) {
        const uint32_t exponent = (j == 3 ? s.s[r] >> 1 : s.s[r] << (23 - 8 * j)) & 0x7f800000u;
        const uint32_t normal = kExact ? normal_exponent<T>(exponent) : exponent;
        const Vec w = from_e2m1<T>(s.w[r][j], __builtin_bit_cast(float, normal)), xv = __builtin_bit_cast(Vec, s.x[j]);
        if constexpr (kExact) {
          const f32x4 d = T::mfma16(xv, w, f32x4{0.f, 0.f, 0.f, 0.f});
          const float rest = __builtin_bit_cast(float, (127u << 23) + exponent - normal);
#pragma unroll
          for (int i = 0; i < kI; i++) acc[r][i] = fmaf(d[i], rest, acc[r][i]);
        } else {
          acc[r] = T::mfma16(xv, w, acc[r]);
        }
      }
  };
  int t = wave;
  Gemv4Step<kR> now, next;
  load(t, now);
  for (; t + waves < a.col_tiles; t += waves) {
    load(t + waves, next);
    multiply(t, now);
    now = next;
  }
  multiply(t, now);
}

constexpr int kMaxWaves = 16;

template <class T, int kR, int kI, class Out>
__global__ __launch_bounds__(64 * (kR == 1 ? kMaxWaves : 8)) void gemv4_kernel(const Gemv4Args a) {
  extern __shared__ __attribute__((aligned(16))) float parts[];  // [waves - 1][kR][kI][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  uint32_t flags[kR], any = 0;
#pragma unroll
  for (int r = 0; r < kR; r++) {
    flags[r] = a.flags[min((int)blockIdx.x * kR + r, a.row_tiles - 1)];
    any |= flags[r];
  }
  f32x4 acc[kR];
#pragma unroll
  for (int r = 0; r < kR; r++) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (any & (T::kIsF16 ? 1u << 16 : 1u << 17))
    gemv4_sum<T, kR, kI, true>(a, acc);
  else
    gemv4_sum<T, kR, kI, false>(a, acc);
  if (wave > 0) {
    float *to = parts + (wave - 1) * (kR * kI * 64) + lane;
#pragma unroll
    for (int r = 0; r < kR; r++)
#pragma unroll
      for (int i = 0; i < kI; i++) to[(r * kI + i) * 64] = acc[r][i];
  }
  if (waves > 1) __syncthreads();
  if (wave > 0) return;
  Out *y = static_cast<Out *>(a.y);
#pragma unroll
  for (int r = 0; r < kR; r++)
#pragma unroll
    for (int i = 0; i < kI; i++) {
      float sum = acc[r][i];
      for (int w = 1; w < waves; w++) sum += parts[(w - 1) * (kR * kI * 64) + (r * kI + i) * 64 + lane];
      if ((flags[r] >> (lane & 15)) & 1) sum = NAN;
      const long long n = ((long long)blockIdx.x * kR + r) * 16 + (lane & 15);
      const int b = 4 * i + (lane >> 4);
      if (n < a.N && b < a.batch) y[b * a.ldy + n] = (Out)sum;
    }
}

// ---- more rows of activations -----------------------------------------------------------
//
// From some rows on the activations are what a CU reads most of, each wave for its own
// tiles. Here a workgroup of 8 waves goes through 4 tiles of rows in chunks of 2 steps of
// 128 columns: activations (8 kX rows), weights and scales of a chunk go straight to LDS,
// the next chunks' in flight meanwhile, a barrier a chunk. A wave takes a tile of one step
// for all rows of activations, so that each weight is converted once; the two steps' sums
// are added up in LDS. Workgroups take groups of tiles in turn, their loads going on from
// one group to the next.
// 37 rows by 12,289 x 8,160: 26 us a call. The kernel alone took 28 when it was taken apart: 7
// remained without loads and products, loads alone added 14 (the activations once for every
// workgroup, 117 MB from L2, beside 53 MB of weights), LDS reads and products 16. With the
// kernel above (four tiles a wave) 31.5, 64 rows 44 against 34. (A wave for two tiles and half
// of the rows: 30.6; for four tiles and 16 rows, each weight converted three times: 36; LDS
// read a chunk ahead of the products: 33; two or four chunks ahead and not three: within 4 %.)
// From 17 rows on, as the kernel above takes no more than 16. Of few tiles of rows most CUs
// have none, and a call takes what calls of 16 rows each would: 16, 17, 32 and 64 rows by
// 4,096 x 4,096 (64 workgroups) 6.3, 11.7, 11.8 and 16.6 us, by 1,024 x 16,384 (16) 18.7, 38, 38
// and 55; of many by 151,936 x 1,024 18.5, 31, 31 and 46.
//
// In LDS a row's 16 bytes c lie at c ^ (row % 16) of the row, so that 16 lanes that read
// one place of 16 rows hit all banks.
constexpr int kTiles = 4, kSteps = 2;

template <int kX>
struct Gemv4Lds {
  static constexpr int kM = (kX + 1) / 2;
  struct Chunk {
    uint8_t x[8 * kX * kSteps * 256], w[kTiles * kSteps * 1024];
    uint32_t s[kTiles * kSteps * 16];
  };
  float parts[kTiles][kM * 4][64];
  static constexpr int kFit = (int)((160 * 1024 - sizeof(parts)) / sizeof(Chunk)), kRing = kFit < 4 ? kFit : 4;
  Chunk chunk[kRing];
};

// 16 (4) bytes for each lane, from `from` and the lane's offset, to LDS in the lanes' order.
// (Inline asm: through the compiler's builtin every later LDS read would wait for all loads
// in flight.)
__device__ __forceinline__ void load_lds16(const void *from, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from), "s"(to)
               : "memory", "m0");
}
__device__ __forceinline__ void load_lds4(const void *from, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(from), "s"(to)
               : "memory", "m0");
}
// Until at most kLeft of the wave's loads are in flight.
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ void gemv4_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
#define SH_GEMV4_LDS __attribute__((address_space(3)))
// A word through the scalar cache (a vector load's wait would be for the chunks in flight).
__device__ __forceinline__ uint32_t constant_word(const uint32_t *p) {
  return *(const __attribute__((address_space(4))) uint32_t *)p;
}

template <class T, int kX, class Out>
__global__ __launch_bounds__(512) void gemv4_rows_kernel(const Gemv4Args a) {
  typedef Gemv4Lds<kX> Lds;
  typedef typename Lds::Chunk Chunk;
  typedef typename T::Vec Vec;
  constexpr int kM = Lds::kM, kRing = Lds::kRing, kRow = kSteps * 256, kPlaces = kSteps * 16;
  constexpr int kXSlots = 4 * kX, kXLoads = (kXSlots + 7) / 8, kLoads = kXLoads + 2;  // (of the wave; KiB of x)
  static_assert(kRing >= 2 && (kRing - 1) * kLoads <= 63, "chunks in flight, and what vmcnt counts");
  __shared__ __attribute__((aligned(16))) Lds lds;
  const int lane = threadIdx.x & 63, r16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = wave % kTiles, step = wave / kTiles;
  const int groups = (a.row_tiles + kTiles - 1) / kTiles, chunks = (a.col_tiles + kSteps - 1) / kSteps;
  const int items = (groups - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x * chunks;
  const uint32_t base = (uint32_t)(uintptr_t)(SH_GEMV4_LDS Chunk *)lds.chunk;

  // the next item (a group's chunk) of this workgroup, requested into the next buffer;
  // behind the last the last again, which nobody reads, so that as many loads are in flight
  int next_group = blockIdx.x, next_chunk = 0, next_buf = 0;
  uint32_t x_row[kXLoads], x_col[kXLoads];  // bytes of the lane's row from x, of its columns from the chunk's first
#pragma unroll
  for (int u = 0; u < kXLoads; u++) {
    const int at = min(wave + 8 * u, kXSlots - 1) * 64 + lane, row = at / kPlaces;
    x_row[u] = (uint32_t)min(row, a.batch - 1) * ((uint32_t)a.ldx * 2);
    x_col[u] = 16 * (at % kPlaces ^ (row & 15));
  }
  auto request = [&]() __attribute__((always_inline)) {
    const int t0 = next_chunk * kSteps, first = next_group * kTiles;
    const uint32_t to = base + next_buf * (uint32_t)sizeof(Chunk), x_last = (uint32_t)(a.K - 8 - 128 * t0) * 2;
    const uint8_t *x = reinterpret_cast<const uint8_t *>(a.x) + (size_t)t0 * 256;
#pragma unroll
    for (int u = 0; u < kXLoads; u++)
      load_lds16(x, x_row[u] + min(x_col[u], x_last), to + offsetof(Chunk, x) + min(wave + 8 * u, kXSlots - 1) * 1024);
    const int tile = min(first + mine, a.row_tiles - 1), t = min(t0 + step, a.col_tiles - 1);
    load_lds16(a.w + ((size_t)tile * a.col_tiles + t) * 1024, lane * 16, to + offsetof(Chunk, w) + wave * 1024);
    // (scales: half of the waves two tiles' two steps each, the others the same)
    const int s_tile = min(first + mine / 2 * 2, a.row_tiles - 1), s_one = min(s_tile + 1, a.row_tiles - 1) - s_tile;
    const int s_step = min(t0 + (grp & 1), a.col_tiles - 1);
    load_lds4(a.scales + (size_t)s_tile * a.col_tiles * 64, ((uint32_t)((grp >> 1) * s_one) * a.col_tiles + s_step) * 64 + r16 * 4,
              to + offsetof(Chunk, s) + mine / 2 * 256);
    next_buf = next_buf + 1 == kRing ? 0 : next_buf + 1;
    if (next_chunk + 1 < chunks)
      next_chunk++;
    else if (next_group + (int)gridDim.x < groups) {
      next_chunk = 0;
      next_group += gridDim.x;
    }
  };

  f32x4 acc[kM];
  int x_at[kM];
#pragma unroll
  for (int m = 0; m < kM; m++) {
    acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int row = min(16 * m + r16, 8 * kX - 1);
    x_at[m] = row * kRow + step * 256 + ((grp ^ (row & 15)) * 16);
  }
  auto compute = [&](const Chunk &c, int t, bool exact) __attribute__((always_inline)) {
    u32x4 x[4][kM];
    const u32x4 w = *reinterpret_cast<const u32x4 *>(c.w + wave * 1024 + lane * 16);
    const uint32_t s = c.s[mine * 32 + step * 16 + r16];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int m = 0; m < kM; m++) x[j][m] = *reinterpret_cast<const u32x4 *>(c.x + (x_at[m] ^ (64 * j)));
    if (128 * t + 128 > a.K) {  // columns behind the last: zeros, whatever x has there
#pragma unroll
      for (int j = 1; j < 4; j++)
#pragma unroll
        for (int m = 0; m < kM; m++)
          if (128 * t + 32 * j >= a.K) x[j][m] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t exponent = (j == 3 ? s >> 1 : s << (23 - 8 * j)) & 0x7f800000u;
      const uint32_t normal = exact ? normal_exponent<T>(exponent) : exponent;
      const Vec wv = from_e2m1<T>(w[j], __builtin_bit_cast(float, normal));
#pragma unroll
      for (int m = 0; m < kM; m++) {
        const Vec xv = __builtin_bit_cast(Vec, x[j][m]);
        if (exact) {
          const f32x4 d = T::mfma16(xv, wv, f32x4{0.f, 0.f, 0.f, 0.f});
          const float rest = __builtin_bit_cast(float, (127u << 23) + exponent - normal);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[m][i] = fmaf(d[i], rest, acc[m][i]);
        } else {
          acc[m] = T::mfma16(xv, wv, acc[m]);
        }
      }
    }
  };

#pragma unroll
  for (int i = 0; i < kRing - 1; i++) request();
  int group = blockIdx.x, chunk = 0, buf = 0;
  uint32_t flags = 0;
  for (int item = 0; item < items; item++) {
    const int t = chunk * kSteps + step;
    if (chunk == 0) flags = constant_word(a.flags + min(group * kTiles + mine, a.row_tiles - 1));
    wait_loads<(kRing - 2) * kLoads>();
    gemv4_barrier();  // every wave's part of the chunk is here, and the last chunk is read
    request();
    if (t < a.col_tiles) {
      if (flags & (T::kIsF16 ? 1u << 16 : 1u << 17))
        compute(lds.chunk[buf], t, true);
      else
        compute(lds.chunk[buf], t, false);
    }
    buf = buf + 1 == kRing ? 0 : buf + 1;
    if (++chunk < chunks) continue;
    chunk = 0;
    if (step == 1) {
#pragma unroll
      for (int m = 0; m < kM; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) lds.parts[mine][4 * m + i][lane] = acc[m][i];
    }
    gemv4_barrier();  // (the parts are read before the next group's last chunk is)
    if (step == 0) {
      Out *y = static_cast<Out *>(a.y);
      const long long n = ((long long)group * kTiles + mine) * 16 + r16;
#pragma unroll
      for (int m = 0; m < kM; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float sum = (flags >> r16) & 1 ? NAN : acc[m][i] + lds.parts[mine][4 * m + i][lane];
          const int b = 16 * m + 4 * grp + i;
          if (n < a.N && b < a.batch) y[b * a.ldy + n] = (Out)sum;
        }
    }
#pragma unroll
    for (int m = 0; m < kM; m++) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    group += gridDim.x;
  }
  wait_loads<0>();  // (nothing is to arrive in LDS that is another workgroup's)
}

// Tiles of rows for a workgroup and waves for its columns (measured in us).
// Few tiles, or little in all: one, and as many waves as there are steps, from 5 rows of x
// on, which each wave reads, 4 where the tiles fill the card. (One row of x by 4,096 x
// 4,096: one tile and 8 waves 4.7, four 6.8; 8 rows by 16,384 x 1,024: one tile and 4 waves 5.6,
// 16 waves 6.4, four tiles 7.6; one row by 8,192 x 4,096 6.9 and 7.1.)
// More: four, with a few steps for a wave. (One row by 12,289 x 8,160: one tile 17.0, four
// 12.1; by 151,936 x 1,024 with one step a wave 23, 2 15.1, 4 15.7, 8 15.8; 16 rows by the same
// 2 steps 22.3, 8 20.4, by 12,289 x 8,160 with 8 waves 19.8, 4 18.0.)
template <class T, int kI, class Out>
hipError_t launch_gemv4(hipStream_t st, const Gemv4Args &a) {
  if (a.row_tiles < 512 || (long long)a.row_tiles * a.col_tiles <= 8192) {
    const int waves = std::min(kI > 1 && a.row_tiles >= 256 ? 4 : kMaxWaves, a.col_tiles);
    gemv4_kernel<T, 1, kI, Out><<<a.row_tiles, 64 * waves, (size_t)(waves - 1) * kI * 256, st>>>(a);
  } else {
    const int waves = kI == 1 ? std::max(1, std::min(8, a.col_tiles / 2)) : std::max(1, std::min(4, a.col_tiles / 8));
    gemv4_kernel<T, 4, kI, Out><<<(a.row_tiles + 3) / 4, 64 * waves, (size_t)(waves - 1) * 4 * kI * 256, st>>>(a);
  }
  return hipGetLastError();
}

template <class T, int kX, class Out>
hipError_t launch_gemv4_rows(hipStream_t st, const Gemv4Args &a) {
  const int groups = (a.row_tiles + kTiles - 1) / kTiles;
  gemv4_rows_kernel<T, kX, Out><<<std::min(groups, 256), 512, 0, st>>>(a);
  return hipGetLastError();
}

template <class T, class Out>
hipError_t launch_gemv4_batch(hipStream_t st, const Gemv4Args &a) {
  if (a.batch <= 4) return launch_gemv4<T, 1, Out>(st, a);
  if (a.batch <= 8) return launch_gemv4<T, 2, Out>(st, a);
  if (a.batch <= 16) return launch_gemv4<T, 4, Out>(st, a);
  if (a.batch <= 24) return launch_gemv4_rows<T, 3, Out>(st, a);
  if (a.batch <= 32) return launch_gemv4_rows<T, 4, Out>(st, a);
  if (a.batch <= 40) return launch_gemv4_rows<T, 5, Out>(st, a);
  if (a.batch <= 48) return launch_gemv4_rows<T, 6, Out>(st, a);
  return launch_gemv4_rows<T, 8, Out>(st, a);
}

template <class T, class Out>
int gemv4(sh_ctx *ctx, const uint16_t *x, int ldx, const uint8_t *w_tiled, Out *y, int ldy, int batch, int K, int N) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (const char *wrong = check_gemv4_sizes(batch, K, N, ldx, ldy)) return fail(SH_ERR_INVALID_ARGUMENT, "gemv_w4a16: %s", wrong);
  if (N == 0) return SH_OK;
  const Gemv4Layout at(N, K);
  const size_t x_bytes = ((size_t)(batch - 1) * ldx + K) * 2, y_bytes = ((size_t)(batch - 1) * ldy + N) * sizeof(Out);
  if ((rc = check_range(ctx, x, x_bytes, "x")) || (rc = check_range(ctx, w_tiled, at.bytes(), "w_tiled")) ||
      (rc = check_range(ctx, y, y_bytes, "y")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w_tiled)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "x and w_tiled must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(y) % sizeof(Out)) return fail(SH_ERR_INVALID_ARGUMENT, "y must be aligned to its values");
  if (ranges_overlap(y, y_bytes, x, x_bytes) || ranges_overlap(y, y_bytes, w_tiled, at.bytes()))
    return fail(SH_ERR_INVALID_ARGUMENT, "y overlaps x or w_tiled");
  Gemv4Args a;
  a.x = x;
  a.w = w_tiled;
  a.scales = w_tiled + at.scales_at();
  a.flags = reinterpret_cast<const uint32_t *>(w_tiled + at.flags_at());
  a.y = y;
  a.batch = batch;
  a.K = K;
  a.N = N;
  a.ldx = ldx;
  a.ldy = ldy;
  a.row_tiles = (int)at.row_tiles;
  a.col_tiles = (int)at.col_tiles;
  typedef typename std::conditional<std::is_same<Out, float>::value, float, typename T::Value>::type Value;
  const hipError_t e = launch_gemv4_batch<T, Value>(stream_of(ctx), a);
  return e == hipSuccess ? SH_OK : hip_fail(e, "gemv_w4a16");
}

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_quantize_e2m1(sh_ctx *ctx, const float *W, int N, int K, uint8_t *q, uint8_t *scales) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (const char *wrong = check_e2m1_sizes(N, K)) return fail(SH_ERR_INVALID_ARGUMENT, "quantize_e2m1: %s", wrong);
  if (N == 0) return SH_OK;
  const size_t groups = (size_t)N * (K / 32);
  if ((rc = check_range(ctx, W, groups * 128, "W")) || (rc = check_range(ctx, q, groups * 16, "q")) ||
      (rc = check_range(ctx, scales, groups, "scales")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(q)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "W and q must be 16-byte aligned");
  if (ranges_overlap(q, groups * 16, W, groups * 128) || ranges_overlap(scales, groups, W, groups * 128) ||
      ranges_overlap(q, groups * 16, scales, groups))
    return fail(SH_ERR_INVALID_ARGUMENT, "q and scales must not overlap W or each other");
  // (a launch takes fewer than 2^32 threads)
  const size_t most = (size_t)1 << 30;
  for (size_t g = 0; g < groups; g += most) {
    const size_t n = std::min(groups - g, most);
    quantize_e2m1_kernel<<<(unsigned)((n + kT - 1) / kT), kT, 0, stream_of(ctx)>>>(W + g * 32, n, q + g * 16, scales + g);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "quantize_e2m1");
}

SH_API int sh_e2m1_tiles_bytes(int N, int K, size_t *bytes) {
  if (!bytes) return fail(SH_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (const char *wrong = check_e2m1_sizes(N, K)) return fail(SH_ERR_INVALID_ARGUMENT, "e2m1_tiles_bytes: %s", wrong);
  *bytes = Gemv4Layout(N, K).bytes();
  return SH_OK;
}

SH_API int sh_pack_e2m1_tiles(sh_ctx *ctx, const uint8_t *q, const uint8_t *scales, int N, int K, uint8_t *tiled) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (const char *wrong = check_e2m1_sizes(N, K)) return fail(SH_ERR_INVALID_ARGUMENT, "pack_e2m1_tiles: %s", wrong);
  if (N == 0) return SH_OK;
  const size_t groups = (size_t)N * (K / 32);
  const Gemv4Layout at(N, K);
  if ((rc = check_range(ctx, q, groups * 16, "q")) || (rc = check_range(ctx, scales, groups, "scales")) ||
      (rc = check_range(ctx, tiled, at.bytes(), "tiled")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(q) & 3) || (reinterpret_cast<uintptr_t>(tiled) & 15))
    return fail(SH_ERR_INVALID_ARGUMENT, "q must be 4-byte and tiled 16-byte aligned");
  if (ranges_overlap(tiled, at.bytes(), q, groups * 16) || ranges_overlap(tiled, at.bytes(), scales, groups))
    return fail(SH_ERR_INVALID_ARGUMENT, "tiled overlaps q or scales");
  // (a launch takes fewer than 2^32 threads)
  const int waves = (int)std::min<size_t>(std::min<size_t>(at.col_tiles, kPackT / 64), ((size_t)1 << 25) / at.row_tiles);
  pack_e2m1_kernel<<<(unsigned)at.row_tiles, 64 * waves, 0, stream_of(ctx)>>>(
      q, scales, N, K, (int)at.col_tiles, tiled, reinterpret_cast<uint32_t *>(tiled + at.scales_at()),
      reinterpret_cast<uint32_t *>(tiled + at.flags_at()));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "pack_e2m1_tiles");
}

SH_API int sh_gemv_w4a16_f16(sh_ctx *ctx, const uint16_t *x, int ldx, const uint8_t *w_tiled, uint16_t *y, int ldy,
                             int batch, int K, int N) {
  return gemv4<PagedF16>(ctx, x, ldx, w_tiled, y, ldy, batch, K, N);
}

SH_API int sh_gemv_w4a16_bf16(sh_ctx *ctx, const uint16_t *x, int ldx, const uint8_t *w_tiled, uint16_t *y, int ldy,
                              int batch, int K, int N) {
  return gemv4<PagedBf16>(ctx, x, ldx, w_tiled, y, ldy, batch, K, N);
}

SH_API int sh_gemv_w4a16_f16_f32(sh_ctx *ctx, const uint16_t *x, int ldx, const uint8_t *w_tiled, float *y, int ldy,
                                 int batch, int K, int N) {
  return gemv4<PagedF16>(ctx, x, ldx, w_tiled, y, ldy, batch, K, N);
}

SH_API int sh_gemv_w4a16_bf16_f32(sh_ctx *ctx, const uint16_t *x, int ldx, const uint8_t *w_tiled, float *y, int ldy,
                                  int batch, int K, int N) {
  return gemv4<PagedBf16>(ctx, x, ldx, w_tiled, y, ldy, batch, K, N);
}

}  // extern "C"
