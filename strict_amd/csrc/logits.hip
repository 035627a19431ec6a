// Rules on rows of logits (sh_adjust_logits_*): penalties for the tokens that a row has
// had, biases and masks.
//
// A workgroup takes kSlice logits of a row. What the row's tokens say of them is counted in
// LDS: a word for each logit, bit 31 where the token is in the prompt, below it how often
// it stands behind (whole numbers: the order of the atomics changes nothing). The
// logits are requested before the tokens are read and go through once; biases, few and
// scattered, are added afterwards to what the workgroup has written.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "paged.h"
#include "sample.h"

namespace sh {
namespace {

constexpr int kT = 512;

struct LogitArgs {
  const void *x;
  float *y;
  size_t ldx, ldy;
  int n, rows;
  sh_logit_rules rules;
};

// Four values that are aligned as one.
template <class V>
struct __attribute__((packed, aligned(sizeof(V)))) Four {
  V v[4];
};

__device__ __forceinline__ float or_else(const float *p, int r, float otherwise) { return p ? p[r] : otherwise; }

// kWhole: all of the slice's logits are there.
template <class V, int kSlice, bool kWhole>
__device__ __forceinline__ void adjust_slice(const LogitArgs &a, uint32_t *table) {
#pragma clang fp contract(off)
  constexpr int kVectors = kSlice / (4 * kT);
  const int row = blockIdx.x, first = blockIdx.y * kSlice, tid = threadIdx.x, n = a.n;
  const sh_logit_rules &rules = a.rules;
  const V *x = static_cast<const V *>(a.x) + row * a.ldx;
  float *y = a.y + row * a.ldy;
  float v[kVectors][4];
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
    const int i = first + 4 * (tid + u * kT);
    if constexpr (kWhole) {
      const Four<V> four = *reinterpret_cast<const Four<V> *>(x + i);
#pragma unroll
      for (int e = 0; e < 4; e++) v[u][e] = (float)four.v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[u][e] = i + e < n ? (float)x[i + e] : 0.0f;
    }
  }
  int length = 0, prompt = 0, bias0 = 0, bias1 = 0, mask = -1;
  if (rules.tokens) {
    length = clamp_int(rules.lengths[row], 0, rules.max_tokens);
    prompt = rules.prompts ? clamp_int(rules.prompts[row], 0, length) : 0;
  }
  if (rules.bias_starts) {
    bias0 = clamp_int(rules.bias_starts[row], 0, rules.bias_count);
    bias1 = clamp_int(rules.bias_starts[row + 1], bias0, rules.bias_count);
  }
  if (rules.masks) mask = rules.mask_of[row];
  if (mask >= rules.num_masks) mask = -1;
  const uint32_t *words = rules.masks + (size_t)max(mask, 0) * ((n + 31) / 32);

  if (length > 0) {
    for (int i = tid; i < kSlice / 4; i += kT) *reinterpret_cast<u32x4 *>(table + 4 * i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    const int32_t *tokens = rules.tokens + (size_t)row * rules.max_tokens;
    const int whole = length & ~3;
    const auto count = [&](int token, int at) {
      const unsigned i = (unsigned)token - (unsigned)first;
      if (i < (unsigned)kSlice && token < n) {  // (first >= 0: no negative token is in a slice)
        if (at >= prompt)
          atomicAdd(&table[i], 1u);
        else
          atomicOr(&table[i], 0x80000000u);
      }
    };
    for (int at = 4 * tid; at < whole; at += 4 * kT) {
      const Four<int32_t> four = *reinterpret_cast<const Four<int32_t> *>(tokens + at);
#pragma unroll
      for (int e = 0; e < 4; e++) count(four.v[e], at + e);
    }
    if (whole + tid < length) count(tokens[whole + tid], whole + tid);
    __syncthreads();
  }
  float repetition = or_else(rules.repetition, row, 1.0f);
  if (!(repetition > 0.0f) || repetition == INFINITY) repetition = 1.0f;
  float frequency = or_else(rules.frequency, row, 0.0f), presence = or_else(rules.presence, row, 0.0f);
  frequency = frequency == frequency ? frequency : 0.0f;
  presence = presence == presence ? presence : 0.0f;
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
    const int at = 4 * (tid + u * kT), i = first + at;
    if (!kWhole && i >= n) continue;
    if (length > 0) {
      const u32x4 t = *reinterpret_cast<const u32x4 *>(table + at);
      if ((t.x | t.y | t.z | t.w) != 0) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (t[e] != 0) v[u][e] = v[u][e] > 0.0f ? v[u][e] / repetition : v[u][e] * repetition;
          const uint32_t c = t[e] & 0x7fffffffu;
          if (c != 0) v[u][e] -= frequency * (float)c + presence;
        }
      }
    }
    if (mask >= 0) {
      const uint32_t bits = words[i >> 5] >> (i & 31);
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (!((bits >> e) & 1)) v[u][e] = -INFINITY;
    }
    if constexpr (kWhole) {
      Four<float> four;
#pragma unroll
      for (int e = 0; e < 4; e++) four.v[e] = v[u][e];
      *reinterpret_cast<Four<float> *>(y + i) = four;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (i + e < n) y[i + e] = v[u][e];
    }
  }
  if (bias0 >= bias1) return;
  // Of a token's biases the last: the largest number of its entries, found in its word.
  const auto place = [&](int e) {
    const int token = rules.bias_tokens[e];
    const unsigned i = (unsigned)token - (unsigned)first;
    return token < n && i < (unsigned)kSlice ? (int)i : -1;
  };
  __syncthreads();  // the table is read, y is written
  for (int e = bias0 + tid; e < bias1; e += kT) {
    const int i = place(e);
    if (i >= 0) table[i] = 0;
  }
  __syncthreads();
  for (int e = bias0 + tid; e < bias1; e += kT) {
    const int i = place(e);
    if (i >= 0) atomicMax(&table[i], (uint32_t)(e - bias0) + 1);
  }
  __syncthreads();
  for (int e = bias0 + tid; e < bias1; e += kT) {
    const int i = place(e), token = first + i;
    if (i < 0 || table[i] != (uint32_t)(e - bias0) + 1) continue;
    if (mask >= 0 && !((words[token >> 5] >> (token & 31)) & 1)) continue;
    y[token] += rules.bias_values[e];
  }
}

template <class V, int kSlice>
__global__ __launch_bounds__(kT) void adjust_logits_kernel(const LogitArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t table[kSlice];
  if ((int)(blockIdx.y + 1) * kSlice <= a.n)
    adjust_slice<V, kSlice, true>(a, table);
  else
    adjust_slice<V, kSlice, false>(a, table);
}

template <class V>
int adjust_logits(sh_ctx *ctx, const void *x, int ldx, float *y, int ldy, int rows, int n, const sh_logit_rules *rules) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (!rules) return fail(SH_ERR_INVALID_ARGUMENT, "rules is NULL");
  if (const char *wrong = check_logits_sizes(rows, n, ldx, ldy, rules)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (rows == 0) return SH_OK;
  const sh_logit_rules &r = *rules;
  const size_t per_row = (size_t)rows * 4, mask_words = (size_t)(n + 31) / 32;
  const size_t x_bytes = ((size_t)(rows - 1) * ldx + n) * sizeof(V), y_bytes = ((size_t)(rows - 1) * ldy + n) * 4;
  if ((rc = check_range(ctx, x, x_bytes, "x")) || (rc = check_range(ctx, y, y_bytes, "y"))) return rc;
  if (reinterpret_cast<uintptr_t>(x) % sizeof(V) || reinterpret_cast<uintptr_t>(y) % 4)
    return fail(SH_ERR_INVALID_ARGUMENT, "x and y must be aligned to their values");
  const bool in_place = x == y && ldx == ldy && sizeof(V) == 4;
  if (!in_place && ranges_overlap(x, x_bytes, y, y_bytes))
    return fail(SH_ERR_INVALID_ARGUMENT, "y overlaps x without being x (fp32, ldy = ldx)");
  const struct {
    const void *p;
    size_t bytes;
    const char *name;
  } used[] = {
      {r.tokens, r.tokens ? (size_t)rows * r.max_tokens * 4 : 0, "tokens"},
      {r.tokens ? r.lengths : nullptr, per_row, "lengths"},
      {r.tokens ? r.prompts : nullptr, per_row, "prompts"},
      {r.repetition, per_row, "repetition"},
      {r.frequency, per_row, "frequency"},
      {r.presence, per_row, "presence"},
      {r.bias_starts, per_row + 4, "bias_starts"},
      {r.bias_starts ? r.bias_tokens : nullptr, (size_t)std::max(r.bias_count, 0) * 4, "bias_tokens"},
      {r.bias_starts ? r.bias_values : nullptr, (size_t)std::max(r.bias_count, 0) * 4, "bias_values"},
      {r.masks, r.masks ? (size_t)r.num_masks * mask_words * 4 : 0, "masks"},
      {r.masks ? r.mask_of : nullptr, per_row, "mask_of"},
  };
  for (const auto &u : used) {
    if (!u.p || u.bytes == 0) continue;
    if ((rc = check_range(ctx, u.p, u.bytes, u.name))) return rc;
    if (reinterpret_cast<uintptr_t>(u.p) & 3)
      return fail(SH_ERR_INVALID_ARGUMENT, "%s must be 4-byte aligned", u.name);
    if (ranges_overlap(u.p, u.bytes, y, y_bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "y overlaps %s", u.name);
  }
  LogitArgs a = {x, y, (size_t)ldx, (size_t)ldy, n, rows, r};
  if (r.max_tokens == 0) a.rules.tokens = nullptr;
  if (r.bias_count == 0) a.rules.bias_starts = nullptr;
  const hipStream_t st = stream_of(ctx);
  if ((long long)rows * ((n + 8191) / 8192) < 512)
    adjust_logits_kernel<V, 2048><<<dim3((unsigned)rows, (unsigned)((n + 2047) / 2048)), kT, 0, st>>>(a);
  else
    adjust_logits_kernel<V, 8192><<<dim3((unsigned)rows, (unsigned)((n + 8191) / 8192)), kT, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "adjust_logits");
}

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_adjust_logits_f32(sh_ctx *ctx, const float *x, int ldx, float *y, int ldy, int rows, int n,
                                const sh_logit_rules *rules) {
  return adjust_logits<float>(ctx, x, ldx, y, ldy, rows, n, rules);
}

SH_API int sh_adjust_logits_f16(sh_ctx *ctx, const uint16_t *x, int ldx, float *y, int ldy, int rows, int n,
                                const sh_logit_rules *rules) {
  return adjust_logits<_Float16>(ctx, x, ldx, y, ldy, rows, n, rules);
}

SH_API int sh_adjust_logits_bf16(sh_ctx *ctx, const uint16_t *x, int ldx, float *y, int ldy, int rows, int n,
                                 const sh_logit_rules *rules) {
  return adjust_logits<__bf16>(ctx, x, ldx, y, ldy, rows, n, rules);
}

}  // extern "C"
