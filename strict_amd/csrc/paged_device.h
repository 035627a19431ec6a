// Device helpers of the operators over a KV cache in pages (paged_ops.hip,
// paged_attn.hip): the two 16-bit types and their conversions, and the pointer
// checks that both files' entry points share.
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
  static constexpr float kWeightLog2 = 7.0f, kMaxScore = 0x1p24f;
  static __device__ __forceinline__ f32x4 mfma16(Vec a, Vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(Vec a, Vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // sum and the eight values, two at a time (fp16 below the normal range as they are)
  static __device__ __forceinline__ float sum8(Vec v, float sum) {
    typedef _Float16 Pair __attribute__((ext_vector_type(2)));
    const Pair one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_fdot2(Pair{v[2 * i], v[2 * i + 1]}, one, sum, false);
    return sum;
  }
};
struct PagedBf16 {
  typedef __bf16 Value;
  typedef pbf16x8 Vec;
  static constexpr float kWeightLog2 = 0.0f, kMaxScore = 0x1p30f;
  static __device__ __forceinline__ f32x4 mfma16(Vec a, Vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(Vec a, Vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // (a step may be off by 2^-23 of the sum)
  static __device__ __forceinline__ float sum8(Vec v, float sum) {
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    const Pair one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_fdot2_f32_bf16(Pair{v[2 * i], v[2 * i + 1]}, one, sum, false);
    return sum;
  }
};

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

inline int check_paged_pointers(sh_ctx *ctx, const sh_paged_kv *kv) {
  int rc;
  const size_t pool = paged_pool_bytes(kv);
  if ((rc = check_range(ctx, kv->k, pool, "k pages")) || (rc = check_range(ctx, kv->v, pool, "v pages")) ||
      (rc = check_range(ctx, kv->page_table, (size_t)kv->batch * kv->max_pages * 4, "page_table")) ||
      (rc = check_range(ctx, kv->lengths, (size_t)kv->batch * 4, "lengths")) ||
      (rc = check_range(ctx, kv->starts, ((size_t)kv->batch + 1) * 4, "starts")))
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

}  // namespace sh
