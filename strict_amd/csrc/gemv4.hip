// Products of a few rows of 16-bit activations with a matrix of 4-bit weights
// (sh_gemv_w4a16_*), and the weights' quantisation and layout.
//
// y[b][n] = sum over groups g of 32 columns of 2^(scale[n][g] - 127) sum_k x[b][k] w[n][k],
// w one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (OCP E2M1, MX scales).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "gemv4.h"
#include "paged.h"
#include "paged_device.h"

namespace sh {
namespace {

constexpr int kT = 256;

// ---- quantisation and layout ---------------------------------------------------------

// A thread a group: the smallest scale 2^e, e >= -127, for which its largest value is at
// most 6 * 2^e = 1.5 * 2^(e + 2), each value to the nearest (half way: the even one).
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
  const float to_group = __builtin_bit_cast(float, e == 127 ? 0x400000u : (uint32_t)(127 - e) << 23);  // 2^-e
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

// A wave takes 16 rows. A group of zeros gets the scale 1, whatever its own.
__global__ __launch_bounds__(64) void pack_e2m1_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ scales,
                                                       int N, int K, int col_tiles, uint8_t *w, uint32_t *tile_scales,
                                                       uint32_t *tile_flags) {
  const int lane = threadIdx.x, r16 = lane & 15, grp = lane >> 4;
  const size_t tile = blockIdx.x, row = tile * 16 + r16;
  const bool there = row < (size_t)N;
  bool nan = false, no_f16 = false, no_bf16 = false;
  for (size_t t = 0; t < (size_t)col_tiles; t++) {
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
  if (lane == 0) tile_flags[tile] = flags;
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

// What a wave has of a step: kR tiles of weights, their scales, and the activations.
template <int kR, int kM>
struct Gemv4Step {
  u32x4 w[kR], x[kM][4];
  uint32_t s[kR];
};

// A workgroup takes kR tiles of rows; its waves share the columns, step by step of 128 in
// turn, and add up in LDS in their order. Activations are the rows of the products, weights
// the columns, so that a lane's results are of one row of weights: 16 kM rows of x, row b
// in the product's row 4 (b % 4) + b / 4, so that up to 4 of them need one register (kI)
// and up to 8 two. Where a scale leaves the type's normal numbers (kExact), weights are
// converted with the nearest that does not, and each group's sum is multiplied by the rest.
template <class T, int kR, int kM, int kI, bool kExact>
__device__ __forceinline__ void gemv4_sum(const Gemv4Args &a, f32x4 (&acc)[kR][kM]) {
  typedef typename T::Vec Vec;
  const int lane = threadIdx.x & 63, r16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const uint16_t *x[kM];
#pragma unroll
  for (int m = 0; m < kM; m++) {
    const int b = 16 * m + 4 * (r16 & 3) + (r16 >> 2);
    x[m] = a.x + (size_t)min(b, a.batch - 1) * a.ldx + grp * 8;
  }
  size_t first[kR];
#pragma unroll
  for (int r = 0; r < kR; r++) first[r] = (size_t)min((int)blockIdx.x * kR + r, a.row_tiles - 1) * a.col_tiles;
  auto load = [&](int t, Gemv4Step<kR, kM> &s) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < kR; r++) {
      s.w[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(a.w + (first[r] + t) * 1024 + lane * 16));
      s.s[r] = *reinterpret_cast<const uint32_t *>(a.scales + (first[r] + t) * 64 + r16 * 4);
    }
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        s.x[m][j] = *reinterpret_cast<const u32x4 *>(x[m] + min(128 * t + 32 * j, a.K - 32));
  };
  auto multiply = [&](int t, Gemv4Step<kR, kM> &s) __attribute__((always_inline)) {
    if (128 * t + 128 > a.K) {  // columns behind the last: zeros, whatever x has there
#pragma unroll
      for (int m = 0; m < kM; m++)
#pragma unroll
        for (int j = 1; j < 4; j++)
          if (128 * t + 32 * j >= a.K) s.x[m][j] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int r = 0; r < kR; r++) {
        uint32_t exponent = (j == 3 ? s.s[r] >> 1 : s.s[r] << (23 - 8 * j)) & 0x7f800000u, rest = 127u << 23;
        if constexpr (kExact) {
          constexpr uint32_t kLeast = T::kIsF16 ? kF16Least : kBf16Least, kMost = T::kIsF16 ? kF16Most : kBf16Most;
          const uint32_t normal = min(max(exponent, kLeast << 23), kMost << 23);
          rest += exponent - normal;
          exponent = normal;
        }
        const Vec w = from_e2m1<T>(s.w[r][j], __builtin_bit_cast(float, exponent));
#pragma unroll
        for (int m = 0; m < kM; m++) {
          const Vec xv = __builtin_bit_cast(Vec, s.x[m][j]);
          if constexpr (kExact) {
            const f32x4 d = T::mfma16(xv, w, f32x4{0.f, 0.f, 0.f, 0.f});
            const float scale = __builtin_bit_cast(float, rest);
#pragma unroll
            for (int i = 0; i < kI; i++) acc[r][m][i] = fmaf(d[i], scale, acc[r][m][i]);
          } else {
            acc[r][m] = T::mfma16(xv, w, acc[r][m]);
          }
        }
      }
  };
  int t = wave;
  if (t >= a.col_tiles) return;
  Gemv4Step<kR, kM> now, next;
  load(t, now);
  for (; t + waves < a.col_tiles; t += waves) {
    load(t + waves, next);
    multiply(t, now);
    now = next;
  }
  multiply(t, now);
}

constexpr int kMaxWaves = 8;

template <class T, int kR, int kM, int kI, class Out>
__global__ __launch_bounds__(64 * kMaxWaves) void gemv4_kernel(const Gemv4Args a) {
  extern __shared__ __attribute__((aligned(16))) float parts[];  // [waves - 1][kR][kM][kI][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  uint32_t flags[kR], any = 0;
#pragma unroll
  for (int r = 0; r < kR; r++) {
    flags[r] = a.flags[min((int)blockIdx.x * kR + r, a.row_tiles - 1)];
    any |= flags[r];
  }
  f32x4 acc[kR][kM];
#pragma unroll
  for (int r = 0; r < kR; r++)
#pragma unroll
    for (int m = 0; m < kM; m++) acc[r][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (any & (T::kIsF16 ? 1u << 16 : 1u << 17))
    gemv4_sum<T, kR, kM, kI, true>(a, acc);
  else
    gemv4_sum<T, kR, kM, kI, false>(a, acc);
  if (wave > 0) {
    float *to = parts + (wave - 1) * (kR * kM * kI * 64) + lane;
#pragma unroll
    for (int r = 0; r < kR; r++)
#pragma unroll
      for (int m = 0; m < kM; m++)
#pragma unroll
        for (int i = 0; i < kI; i++) to[((r * kM + m) * kI + i) * 64] = acc[r][m][i];
  }
  if (waves > 1) __syncthreads();
  if (wave > 0) return;
  Out *y = static_cast<Out *>(a.y);
#pragma unroll
  for (int r = 0; r < kR; r++)
#pragma unroll
    for (int m = 0; m < kM; m++)
#pragma unroll
      for (int i = 0; i < kI; i++) {
        float sum = acc[r][m][i];
        for (int w = 1; w < waves; w++) sum += parts[(w - 1) * (kR * kM * kI * 64) + ((r * kM + m) * kI + i) * 64 + lane];
        if ((flags[r] >> (lane & 15)) & 1) sum = NAN;
        const long long n = ((long long)blockIdx.x * kR + r) * 16 + (lane & 15);
        const int b = 16 * m + 4 * i + (lane >> 4);
        if (n < a.N && b < a.batch) y[b * a.ldy + n] = (Out)sum;
      }
}

template <class T, int kR, int kM, int kI, class Out>
hipError_t launch_gemv4(hipStream_t st, const Gemv4Args &a) {
  const int groups = (a.row_tiles + kR - 1) / kR;
  const int waves = std::max(1, std::min({kMaxWaves, a.col_tiles, 8192 / groups}));
  gemv4_kernel<T, kR, kM, kI, Out><<<groups, 64 * waves, (size_t)(waves - 1) * kR * kM * kI * 256, st>>>(a);
  return hipGetLastError();
}

template <class T, class Out>
hipError_t launch_gemv4_batch(hipStream_t st, const Gemv4Args &a) {
  if (a.batch <= 4) return launch_gemv4<T, 2, 1, 1, Out>(st, a);
  if (a.batch <= 8) return launch_gemv4<T, 2, 1, 2, Out>(st, a);
  if (a.batch <= 16) return launch_gemv4<T, 2, 1, 4, Out>(st, a);
  if (a.batch <= 32) return launch_gemv4<T, 2, 2, 4, Out>(st, a);
  if (a.batch <= 48) return launch_gemv4<T, 2, 3, 4, Out>(st, a);
  return launch_gemv4<T, 2, 4, 4, Out>(st, a);
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
  pack_e2m1_kernel<<<(unsigned)at.row_tiles, 64, 0, stream_of(ctx)>>>(
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
