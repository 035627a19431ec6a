// Rules on rows of logits (sh_adjust_logits_*): penalties for the tokens that a row has
// had, biases and masks.
//
// A workgroup takes kSlice logits of a row. What there is to know of them it gathers in LDS,
// a word for each: bit 31 where the token is in the row's prompt, bit 30 where it has a
// bias, below them how often it stands behind the prompt (whole numbers: the order of the
// atomics changes nothing). The logits are requested before any of that and go through
// once; a biased one is written by the thread that holds its bias. No barrier waits for
// memory. Bound by the bytes: 200 rows of 151,936 logits in bf16 without rules (182 MB) take
// 27.8 us, 6.5 TB/s, with up to 4,000 tokens a row 32, with those, 100 biases and a third of the
// rows masked 37. (Stores that the caches keep: 40 without rules.)
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
struct FourOf {
  typedef V Type __attribute__((ext_vector_type(4), aligned(sizeof(V))));
};
template <class V>
using Four = typename FourOf<V>::Type;

__device__ __forceinline__ float or_else(const float *p, int r, float otherwise) { return p ? p[r] : otherwise; }

__device__ __forceinline__ void lds_barrier() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): loads from memory stay in flight
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

constexpr uint32_t kPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = kBiased - 1;

// A row's penalties, and what they make of a logit whose word is t.
struct Penalties {
  float repetition, frequency, presence;
  __device__ __forceinline__ Penalties(const sh_logit_rules &r, int row)
      : repetition(or_else(r.repetition, row, 1.0f)),
        frequency(or_else(r.frequency, row, 0.0f)),
        presence(or_else(r.presence, row, 0.0f)) {
    if (!(repetition > 0.0f) || repetition == INFINITY) repetition = 1.0f;
    frequency = frequency == frequency ? frequency : 0.0f;
    presence = presence == presence ? presence : 0.0f;
  }
  __device__ __forceinline__ float operator()(float v, uint32_t t) const {
#pragma clang fp contract(off)
    const uint32_t c = t & kCount;
    if ((t & kPrompt) || c != 0) v = v > 0.0f ? v / repetition : v * repetition;
    if (c != 0) v -= frequency * (float)c + presence;
    return v;
  }
};

// kWhole: all of the slice's logits are there.
template <class V, int kSlice, bool kWhole>
__device__ __forceinline__ void adjust_slice(const LogitArgs &a, uint32_t *table) {
#pragma clang fp contract(off)
  constexpr int kVectors = kSlice / (4 * kT);
  const int row = blockIdx.x, first = blockIdx.y * kSlice, tid = threadIdx.x, n = a.n;
  const sh_logit_rules &rules = a.rules;
  const V *x = static_cast<const V *>(a.x) + row * a.ldx;
  float *y = a.y + row * a.ldy;
  V v[kVectors][4];
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
    const int i = first + 4 * (tid + u * kT);
    if constexpr (kWhole) {
      const Four<V> four = *reinterpret_cast<const Four<V> *>(x + i);
#pragma unroll
      for (int e = 0; e < 4; e++) v[u][e] = four[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[u][e] = i + e < n ? x[i + e] : (V)0.0f;
    }
  }
  // (of the row's tokens those that the thread counts first, before it is known whether there
  // are as many)
  const int32_t *tokens = rules.tokens + (size_t)row * rules.max_tokens;
  Four<int32_t> soon = 0;
  if (rules.tokens && 4 * tid + 4 <= rules.max_tokens) soon = *reinterpret_cast<const Four<int32_t> *>(tokens + 4 * tid);
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
  uint32_t allowed[kVectors];
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
    const int i = first + 4 * (tid + u * kT);
    allowed[u] = mask >= 0 && (kWhole || i < n) ? words[i >> 5] >> (i & 31) : 0xf;
  }
  const auto place = [&](int token) {  // in the slice, or -1 (first >= 0: no negative token is)
    const unsigned i = (unsigned)token - (unsigned)first;
    return token < n && i < (unsigned)kSlice ? (int)i : -1;
  };
  // A bias a thread, if there are no more: the last of a token's, the one with the largest
  // number, marks the word; its thread writes the logit.
  const bool few = bias1 - bias0 <= kT;
  int mine = -1;
  float my_bias = 0.0f, my_x = 0.0f;
  if (few && bias0 + tid < bias1) {
    mine = place(rules.bias_tokens[bias0 + tid]);
    if (mine >= 0) {
      my_bias = rules.bias_values[bias0 + tid];
      my_x = (float)x[first + mine];
    }
  }
  const bool gather = length > 0 || (few && bias0 < bias1);
  if (gather) {
    for (int i = tid; i < kSlice / 4; i += kT) *reinterpret_cast<u32x4 *>(table + 4 * i) = u32x4{0, 0, 0, 0};
    lds_barrier();
  }
  if (few && bias0 < bias1) {
    if (mine >= 0) atomicMax(&table[mine], (uint32_t)tid + 1);
    lds_barrier();
    if (mine >= 0 && table[mine] != (uint32_t)tid + 1) mine = -1;
    lds_barrier();
    if (mine >= 0) table[mine] = kBiased;
    lds_barrier();
  }
  if (length > 0) {
    const int whole = length & ~3;
    const auto count = [&](int token, int at) {
      const int i = place(token);
      if (i < 0) return;
      if (at >= prompt)
        atomicAdd(&table[i], 1u);
      else
        atomicOr(&table[i], kPrompt);
    };
    for (int at = 4 * tid; at < whole; at += 4 * kT) {
      const Four<int32_t> four = at == 4 * tid ? soon : *reinterpret_cast<const Four<int32_t> *>(tokens + at);
#pragma unroll
      for (int e = 0; e < 4; e++) count(four[e], at + e);
    }
    if (whole + tid < length) count(tokens[whole + tid], whole + tid);
    lds_barrier();
  }
  const Penalties penalised(rules, row);
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
    const int at = 4 * (tid + u * kT), i = first + at;
    if (!kWhole && i >= n) continue;
    Four<float> out;
#pragma unroll
    for (int e = 0; e < 4; e++) out[e] = (float)v[u][e];
    uint32_t words_of = 0;
    if (gather) {
      const u32x4 t = *reinterpret_cast<const u32x4 *>(table + at);
      words_of = t.x | t.y | t.z | t.w;
      if (words_of != 0) {
#pragma unroll
        for (int e = 0; e < 4; e++) out[e] = penalised(out[e], t[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (!((allowed[u] >> e) & 1)) out[e] = -INFINITY;
    if (kWhole && !(words_of & kBiased)) {
      __builtin_nontemporal_store(out, reinterpret_cast<Four<float> *>(y + i));
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (i + e < n && !(words_of != 0 && (table[at + e] & kBiased))) y[i + e] = out[e];
    }
  }
  const auto ruled_out = [&](int token) { return mask >= 0 && !((words[token >> 5] >> (token & 31)) & 1); };
  if (mine >= 0) y[first + mine] = ruled_out(first + mine) ? -INFINITY : penalised(my_x, table[mine]) + my_bias;
  if (few) return;
  // More biases than threads: the last of each token adds its value to what is written.
  __syncthreads();  // (the table is read, y is written)
  const auto each_bias = [&](auto f) __attribute__((always_inline)) {
    for (int e = bias0 + tid; e < bias1; e += kT) {
      const int i = place(rules.bias_tokens[e]);
      if (i >= 0) f(i, e);
    }
    __syncthreads();
  };
  each_bias([&](int i, int) { table[i] = 0; });
  each_bias([&](int i, int e) { atomicMax(&table[i], (uint32_t)(e - bias0) + 1); });
  each_bias([&](int i, int e) {
    if (table[i] == (uint32_t)(e - bias0) + 1 && !ruled_out(first + i)) y[first + i] += rules.bias_values[e];
  });
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
  // Few rows in small slices, side by side; rows of many tokens, which every slice of the row
  // reads, in large ones. (us with slices of 2,048, 4,096 and 8,192: 20 rows of 151,936 of up to
  // 4,000 tokens 8.7, 6.5, -; 200 -, 36.9, 36.0; of up to 20,000 tokens -, 54.8, 48.8.)
  const auto slices = [&](int slice) { return dim3((unsigned)rows, (unsigned)((n + slice - 1) / slice)); };
  if ((long long)rows * slices(4096).y < 256)
    adjust_logits_kernel<V, 2048><<<slices(2048), kT, 0, st>>>(a);
  else if (!a.rules.tokens || r.max_tokens <= 4096)
    adjust_logits_kernel<V, 4096><<<slices(4096), kT, 0, st>>>(a);
  else
    adjust_logits_kernel<V, 8192><<<slices(8192), kT, 0, st>>>(a);
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
