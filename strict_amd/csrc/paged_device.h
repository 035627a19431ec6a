// Device helpers of the operators over a KV cache in pages (paged_ops.hip,
// paged_attn.hip and their counterparts for pages of 8-bit values): the two 16-bit
// types and their conversions, those from the 8-bit type, a token's sequence and angles,
// and the pointer checks that the entry points share.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"
#include "paged.h"

namespace sh {

typedef _Float16 pf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pbf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// (bf16's range is fp32's, so its weights need no scale; fp16 weights are kept
// 2^7 times as large, which leaves those down to 2^-21 normal and those of a
// maximum that lags behind by up to 2^8 finite.)
// kMaxScore: a row's maximum is q.k scale rounded to fp32, its weights are 2 to the power
// of the unrounded products less that: all are off by one factor, which the division
// takes out again, of up to 2^(half a step of the maximum). Below 2^24 that is 2^(1/2): the
// weights of fp16 stay below 2^15.5, and the maximum less 7 is exact. Below 2^30 it is
// 2^32, which bf16's range has room for. Beyond, weights overflow or all come to 0.
struct PagedF16 {
  typedef _Float16 Value;
  typedef pf16x8 Vec;
  typedef _Float16 Pair __attribute__((ext_vector_type(2)));
  static constexpr bool kIsF16 = true;
  static constexpr float kWeightLog2 = 7.0f, kMaxScore = 0x1p24f;
  static __device__ __forceinline__ f32x4 mfma16(Vec a, Vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(Vec a, Vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // sum and the eight values, two at a time (fp16 below the normal range as they are)
  static __device__ __forceinline__ float sum8(Vec v, float sum) {
    const Pair one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_fdot2(Pair{v[2 * i], v[2 * i + 1]}, one, sum, false);
    return sum;
  }
};
struct PagedBf16 {
  typedef __bf16 Value;
  typedef pbf16x8 Vec;
  typedef __bf16 Pair __attribute__((ext_vector_type(2)));
  static constexpr bool kIsF16 = false;
  static constexpr float kWeightLog2 = 0.0f, kMaxScore = 0x1p30f;
  static __device__ __forceinline__ f32x4 mfma16(Vec a, Vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(Vec a, Vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // (a step may be off by 2^-23 of the sum)
  static __device__ __forceinline__ float sum8(Vec v, float sum) {
    const Pair one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_fdot2_f32_bf16(Pair{v[2 * i], v[2 * i + 1]}, one, sum, false);
    return sum;
  }
};

// Four values of OCP E4M3 (a byte each) times a power of two, in the 16-bit type: exact
// but for what leaves that type's range, rounded as ever. Of `scale` only the exponent
// counts, as an E8M0 byte in its place would: 0 is 2^-127, 255 gives NaN.
__device__ __forceinline__ float e8m0_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
template <class T>
__device__ __forceinline__ u32x2 from_e4m3(uint32_t four, float scale) {
  if constexpr (T::kIsF16)
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(four, scale, true))};
  else
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, true))};
}
template <class T>
__device__ __forceinline__ u32x4 from_e4m3(uint32_t first, uint32_t second, float scale) {
  const u32x2 a = from_e4m3<T>(first, scale), b = from_e4m3<T>(second, scale);
  return u32x4{a.x, a.y, b.x, b.y};
}

template <class T>
__device__ __forceinline__ void unpack8(u32x4 bits, float (&x)[8]) {
  const typename T::Vec v = __builtin_bit_cast(typename T::Vec, bits);
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = (float)v[e];
}

template <class T>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  typename T::Vec v;
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = (typename T::Value)x[e];
  return __builtin_bit_cast(u32x4, v);
}

// cos and sin of an fp64 angle below 2^29 (check_rope_theta) to within 2^-38: reduction by
// pi / 2 in two parts (Cody and Waite) and Taylor polynomials on [-pi / 4, pi / 4], in fp64.
template <class Real>
__device__ __forceinline__ void cos_sin64(double a, Real *c, Real *s) {
  const double q = rint(a * 0.63661977236758134308);  // 2 / pi
  double r = fma(-q, 1.57079632679489655800, a);      // pi / 2 as the nearest double
  r = fma(-q, 6.12323399573676603587e-17, r);         // and the rest
  const double z = r * r;
  // to r^13 / 13! and r^12 / 12!: the next terms are below 2^-38
  double ps = fma(z, 1.60590438368216145994e-10, -2.50521083854417187751e-8);
  ps = fma(z, ps, 2.75573192239858906526e-6);
  ps = fma(z, ps, -1.98412698412698412698e-4);
  ps = fma(z, ps, 8.33333333333333333333e-3);
  ps = fma(z, ps, -1.66666666666666666667e-1);
  const double sr = fma(r * z, ps, r);
  double pc = fma(z, 2.08767569878680989792e-9, -2.75573192239858906526e-7);
  pc = fma(z, pc, 2.48015873015873015873e-5);
  pc = fma(z, pc, -1.38888888888888888889e-3);
  pc = fma(z, pc, 4.16666666666666666667e-2);
  pc = fma(z, pc, -5.0e-1);
  const double cr = fma(z, pc, 1.0);
  const int k = (int)q & 3;
  const double sd = (k & 1) ? cr : sr, cd = (k & 1) ? sr : cr;
  *s = (Real)((k & 2) ? -sd : sd);
  *c = (Real)((k == 1 || k == 2) ? -cd : cd);
}

// A lane's part of a head, kD / 16 lanes wide: y = x / sqrt(mean x^2 + eps) * gain, rotated
// by halves, with factor(e) the cosine and sine of pair e. Which products are fused is
// written out, so that every operator that takes this gives the same bits: left to the
// compiler, one value in 10^4 came out a step of fp16 off between two kernels. (The last
// one's rounding to fp16 is that instruction's own, one rounding and not two: the Makefile
// has these files compiled so that it is everywhere.)
template <int kD, class Factor>
__device__ __forceinline__ void head_norm_rope(float (&x1)[8], float (&x2)[8], const float *gain, float eps, Factor factor) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
#pragma unroll
  for (int off = 1; off < kD / 16; off *= 2) ss += __shfl_xor(ss, off, 64);
  const float inv = 1.0f / sqrtf(fmaf(ss, 1.0f / kD, eps));
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float2 f = factor(e);
    const float y1 = x1[e] * inv * gain[e], y2 = x2[e] * inv * gain[e + kD / 2];
    x1[e] = fmaf(y1, f.x, -(y2 * f.y));
    x2[e] = fmaf(y2, f.x, y1 * f.y);
  }
}

// The sequence that row `row` belongs to: the last b with starts[b] <= row (b =
// batch: behind the last, -1: before the first). A wave looks at 64 values at a
// time; batches of up to 63 take one round.
__device__ __forceinline__ int find_seq(const int *__restrict__ starts, int batch, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = batch + 1;  // the answer is in lo - 1 .. lo + n - 1
  while (true) {
    const int step = (n + 63) / 64, at = lane * step;
    const int below = __popcll(__ballot(at < n && starts[lo + min(at, n - 1)] <= row));
    if (below == 0) return lo - 1;  // (lo > 0 only after starts[lo] <= row was seen)
    lo += (below - 1) * step;
    n = min(step, n - (below - 1) * step);
    if (step == 1) return lo;
  }
}

// The page table, lengths and starts lie in the context's memory, and so that whole integers
// are read: loads at places which a wave shares leave the address's last two bits out.
inline int check_paged_index(sh_ctx *ctx, const sh_paged_kv *kv) {
  int rc;
  if ((rc = check_range(ctx, kv->page_table, (size_t)kv->batch * kv->max_pages * 4, "page_table")) ||
      (rc = check_range(ctx, kv->lengths, (size_t)kv->batch * 4, "lengths")) ||
      (rc = check_range(ctx, kv->starts, ((size_t)kv->batch + 1) * 4, "starts")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(kv->page_table) | reinterpret_cast<uintptr_t>(kv->lengths) |
       reinterpret_cast<uintptr_t>(kv->starts)) & 3)
    return fail(SH_ERR_INVALID_ARGUMENT, "page_table, lengths and starts must be 4-byte aligned");
  return SH_OK;
}

inline int check_paged_pointers(sh_ctx *ctx, const sh_paged_kv *kv) {
  int rc;
  const size_t pool = paged_pool_bytes(kv);
  if ((rc = check_range(ctx, kv->k, pool, "k pages")) || (rc = check_range(ctx, kv->v, pool, "v pages")) ||
      (rc = check_paged_index(ctx, kv)))
    return rc;
  if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "k and v pages must be 16-byte aligned");
  return SH_OK;
}

// Whether [p, p + bytes), which a call writes, lies over what it reads to find its way:
// workgroups that read it before and after would not divide the call alike.
inline bool overlaps_index(const sh_paged_kv *kv, const void *p, size_t bytes) {
  const size_t batch = kv->batch;
  return ranges_overlap(p, bytes, kv->page_table, batch * kv->max_pages * 4) ||
         ranges_overlap(p, bytes, kv->lengths, batch * 4) || ranges_overlap(p, bytes, kv->starts, (batch + 1) * 4);
}

inline int check_paged8_pointers(sh_ctx *ctx, const sh_paged_kv8 *kv) {
  int rc;
  const sh_paged_kv index = paged8_index(kv);
  if ((rc = check_range(ctx, kv->pages, paged8_pool_bytes(kv), "pages")) || (rc = check_paged_index(ctx, &index)))
    return rc;
  if (reinterpret_cast<uintptr_t>(kv->pages) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "pages must be 16-byte aligned");
  return SH_OK;
}

}  // namespace sh
