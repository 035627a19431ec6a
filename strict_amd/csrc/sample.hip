// One token per row of logits by temperature, top-k, top-p and min-p
// (sh_sample_f32; the definition is in strict_hip.h).
//
// A token's weight is exp(-(max - x) / temperature) = 2^-t as a whole number of
// 2^-42: sums of weights are then exact in 64 bits (at most 2^20 tokens), in any
// order, and atomics in any order give the same. The order of the tokens is that
// of 64-bit keys: the value's order above, the complement of the index below.
//
// Rows of up to 2,048 logits, which the list holds: one kernel, one workgroup a row (64
// rows of 2,048 logits 23 us, by the four kernels 34; of 1,000 20 and 24). Longer ones in
// four kernels over (row, split). 200 rows of 151,936: max 19 us, the HBM rate; bins 25
// where top-k ends the selection (an LDS atomic a logit), 44 where top-p does (a weight in
// fp64, too); gather 28 at top-k 50, 35 at 1,000, 47 to 54 where most logits are weighed;
// draw, whose steps wait for each other in one workgroup a row, 7 at top-k 50, 18 at
// 1,000, 20 at top-p 0.95, 27 where rows have several of them. One row of 50,257: 16.5 to
// 18 us, four launches.
//   max     the splits' largest values; clears the row's histogram
//   bins    count of the tokens by t in bins of 1/46, or their weight, where top-p is
//           without top-k; other rows pass
//   gather  from the bins, the bin where top-k (without it, top-p) ends. Up to
//           2,048 tokens to that bin's end: all of them to a list, from which the
//           rest is decided. More: only that bin's tokens, and the weight of the
//           kept tokens before them in each run of 512. Without top-k and top-p: that
//           of all tokens
//   draw    a workgroup a row: ends the selection within the list, finds the run and
//           in it the token that u falls on
// A list that would not hold the bin's tokens, or top-p after a top-k of more than
// the list holds: the draw kernel finds the last kept key by its digits, reading
// the row once per digit: a cliff (200 rows of 151,936 at temperature 40: top-k 50,000 or
// top-p 0.5 1.1 ms, top-k 50,000 with top-p 0.9 2.0; one row 0.6 and 1.1).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "paged.h"
#include "sample.h"

namespace sh {
namespace {

constexpr int kT = 512;
constexpr int kBins = 2048, kBinsPerUnit = 46;
constexpr int kList = 2048;
constexpr int kFraction = 42;       // bits of a weight
constexpr float kCutoff = 43.1f;    // 2^-t 2^42 is below 1/2 from t = 43 on
constexpr int kSegment = 256;       // tokens that a wave takes at once
constexpr int kMaxSegments = kMaxSampleN / kSegment;
constexpr int kRun = 2 * kSegment;  // of the gathering kernel
constexpr int kMaxRuns = kMaxSampleN / kRun;
constexpr int kMaxSplits = 64;

enum { kAll = 0, kListed = 1, kBinned = 2, kDigits = 3 };

// A row's state between the kernels, in the work buffer.
struct RowState {
  unsigned long long mass[kBins];  // weights of the bin's tokens
  unsigned int count[kBins];
  unsigned long long list[kList];  // keys
  unsigned long long run_mass[kMaxRuns];  // weight of the kept tokens before `bin`
  float split_max[kMaxSplits];
  unsigned int listed;
  int mode, bin;                   // bin: where the list ends (kAll: past all bins)
  unsigned int before_count;       // of the tokens in the bins before `bin`
  unsigned long long before_mass;
  unsigned long long limit;        // top-p's, 0: none (or, with top-k, not known yet)
  int k;                           // top-k's, 0: none
};

struct SampleArgs {
  const float *x, *temperature, *top_p, *min_p, *u;
  const int *top_k;
  int *index;
  RowState *rows;
  int n, ld, splits, chunk;
  double table[64];  // 2^(-j / 64)
};

struct RowParams {
  float m;          // largest logit
  float half_m;
  double inv_t;     // log2(e) / temperature
  float inv_2t;     // twice that in fp32
  bool greedy;
  int k;            // 0: all
  double p, least;  // p >= 1: all; least <= 0: all
};

__device__ __forceinline__ RowParams row_params(const SampleArgs &a, int row, float m) {
  RowParams r;
  const float t = a.temperature ? a.temperature[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.0f, least = a.min_p ? a.min_p[row] : 0.0f;
  r.m = m;
  r.greedy = !(t > 0.0f) || k == 1;
  r.half_m = 0.5f * m;
  r.inv_t = 1.4426950408889634074 / (double)t;
  r.inv_2t = fminf((float)(2.0 * r.inv_t), 3.40282347e+38f);
  r.k = k > 0 && k < a.n ? k : 0;
  r.p = p < 1.0f ? (double)p : 1.0;
  r.least = least > 0.0f ? (double)fminf(least, 1.0f) : 0.0;
  return r;
}

// t of a logit to fp32 (NaN for one that is NaN): descends with the logit, which is
// all that the bins need. (Halves, as the difference may exceed fp32's range.)
__device__ __forceinline__ float exponent(const RowParams &r, float x) {
  return x == r.m ? 0.0f : (r.half_m - 0.5f * x) * r.inv_2t;
}

// 2^-t, 0 <= t: t = n / 64 + f, the table's 2^-((n % 64) / 64) and a polynomial of f,
// |f| <= 1 / 128 (next term 4e-17).
__device__ __forceinline__ double exp_minus(double t, const double *table) {
  const double n = rint(t * 64.0), f = fma(n, -1.0 / 64.0, t);
  double e = fma(f, -1.33335581464284434e-3, 9.61812910762847716e-3);  // ln(2)^k / k!
  e = fma(f, e, -5.55041086648215800e-2);
  e = fma(f, e, 2.40226506959100712e-1);
  e = fma(f, e, -6.93147180559945309e-1);
  e = fma(f, e, 1.0);
  const int i = (int)n;
  return ldexp(e * table[i & 63], -(i >> 6));
}

// A logit's weight; *kept: whether min_p keeps it. 0: never drawn.
__device__ __forceinline__ unsigned long long weight(const RowParams &r, float x, const double *table, bool *kept) {
  const double e = exp_minus(x == r.m ? 0.0 : ((double)r.m - (double)x) * r.inv_t, table);
  *kept = e >= r.least;
  // 2^52 + w has w in its low bits, rounded to the nearest
  const double w = fma(e, (double)(1LL << kFraction), 4503599627370496.0);
  return __builtin_bit_cast(unsigned long long, w) & ((1ULL << 52) - 1);
}

__device__ __forceinline__ int bin_of(float t) { return (int)(t * (float)kBinsPerUnit); }

// Order of (value, index), descending; -0 as +0. 0 is no token's key (the value
// of key 0 would be a NaN).
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ int key_index(unsigned long long key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __builtin_bit_cast(float, (u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Logits i .. i + 3 of a row (-infinity from `end` on).
__device__ __forceinline__ f32x4 load4(const float *x, int i, int end) {
  if (i + 4 <= end) return *reinterpret_cast<const f32x4_any *>(x + i);
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = i + e < end ? x[i + e] : -INFINITY;
  return v;
}

template <int kCtrl, int kRowMask>
__device__ __forceinline__ unsigned long long dpp_u64(unsigned long long v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, kRowMask, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), kCtrl, kRowMask, 0xf, false);
  return ((unsigned long long)hi << 32) | lo;
}

// Inclusive sum over the wave's lanes (row_shr:1, 2, 4, 8, row_bcast:15, 31; a lane
// that gets nothing gets 0): a fifth of the time of LDS permutes.
__device__ __forceinline__ unsigned long long wave_scan_u64(unsigned long long v) {
  v += dpp_u64<0x111, 0xf>(v);
  v += dpp_u64<0x112, 0xf>(v);
  v += dpp_u64<0x114, 0xf>(v);
  v += dpp_u64<0x118, 0xf>(v);
  v += dpp_u64<0x142, 0xa>(v);
  v += dpp_u64<0x143, 0xc>(v);
  return v;
}

// Inclusive sum over the workgroup's threads; *total: of all.
__device__ __forceinline__ unsigned long long block_scan_u64(unsigned long long v, unsigned long long *red,
                                                             unsigned long long *total) {
  const int wave = threadIdx.x >> 6;
  v = wave_scan_u64(v);
  __syncthreads();  // red's earlier readers are done
  if ((threadIdx.x & 63) == 63) red[wave] = v;
  __syncthreads();
  unsigned long long sum = 0;
#pragma unroll
  for (int w = 0; w < kT / 64; w++) {
    if (w == wave) v += sum;
    sum += red[w];
  }
  *total = sum;
  return v;
}

__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kT / 64; w++) v = fmaxf(v, red[w]);
  return v;
}

__device__ __forceinline__ unsigned long long block_min_u64(unsigned long long v, unsigned long long *red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const unsigned long long o = __shfl_xor(v, off, 64);
    v = o < v ? o : v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kT / 64; w++) v = red[w] < v ? red[w] : v;
  return v;
}

// Weights before p of the total: the smallest whole number not below.
__device__ __forceinline__ unsigned long long limit_of(double p, unsigned long long total) {
  const double l = ceil(p * (double)total);
  return l >= 1.0 ? (unsigned long long)l : 1ULL;  // (at least one token)
}

// What the weights up to a token must exceed for u to fall on it or before.
__device__ __forceinline__ unsigned long long target_of(const SampleArgs &a, int row, unsigned long long total) {
  const float u = a.u[row];
  const unsigned long long t = u > 0.0f ? (unsigned long long)((double)fminf(u, 1.0f) * (double)total) : 0ULL;
  return t < total ? t : total - 1;
}

// ---- the list of candidates, in LDS ------------------------------------------------

struct Candidates {
  unsigned long long key[kList], mass[kList];
  unsigned long long bucket[1024];  // weights by ten bits of the index, or of the key
  unsigned int held[1024];          // tokens by ten bits of the key
  unsigned int high, low;
};

__device__ __forceinline__ unsigned long long key_weight(const RowParams &r, unsigned long long key,
                                                         const double *table, bool *kept) {
  const float x = key_value(key);
  return weight(r, x, table, kept);
}

__device__ __forceinline__ void weigh_candidates(const RowParams &r, Candidates &c, int n, const double *table) {
  bool kept;
  for (int i = threadIdx.x; i < n; i += kT) c.mass[i] = key_weight(r, c.key[i], table, &kept);
  __syncthreads();
}

// The first of n keys, descending, at which `before` and the keys' counts (by_mass
// false) or weights up to it and with it reach `limit`, which all of them do. By ten
// bits of the keys at a time, from the first in which they differ on, until one key is
// left: two or three rounds mostly, where a sort of 2,048 keys took 66 passes (16 rows
// of 151,936 with top-k 1,000 and top-p 48 -> 40 us a call). Up to 256 keys are compared
// with each other (top-k 50: 26 us, by rounds 30).
constexpr int kCounted = 256;
__device__ __forceinline__ unsigned long long last_key(Candidates &c, int n, bool by_mass, unsigned long long before,
                                                       unsigned long long limit, unsigned long long *red) {
  __syncthreads();  // the last buckets are read
  if (n <= kCounted) {  // each key's sum by itself
    if (((int)threadIdx.x & ~63) < n) {
      const int mine = min((int)threadIdx.x, n - 1);
      const unsigned long long key = c.key[mine], own = by_mass ? c.mass[mine] : 1;
      unsigned long long sum = before;
#pragma unroll 8
      for (int i = 0; i < n; i++) sum += c.key[i] >= key ? (by_mass ? c.mass[i] : 1) : 0;
      if (sum >= limit && sum - own < limit) c.bucket[0] = key;
    }
    __syncthreads();
    return c.bucket[0];
  }
  if (threadIdx.x == 0) {
    c.high = 0;
    c.low = ~0u;
  }
  __syncthreads();
  unsigned high = 0, low = ~0u;
  for (int i = threadIdx.x; i < n; i += kT) {
    const unsigned value = (unsigned)(c.key[i] >> 32);
    high = max(high, value);
    low = min(low, value);
  }
  if (high >= low) {  // (the thread has a key)
    atomicMax(&c.high, high);
    atomicMin(&c.low, low);
  }
  __syncthreads();
  high = c.high;
  const unsigned differ = high ^ c.low;
  // the keys from bit `known` on are `prefix`, the next digit starts at `shift` (of one
  // value: the keys' lower halves are complements of numbers below 2^20)
  int known = differ != 0 ? 64 - __clz(differ) : 20, shift = known - 10;
  unsigned long long prefix =
      known < 64 ? (((unsigned long long)high << 32) | (differ != 0 ? 0u : ~0u)) >> known : 0;
  while (true) {
    for (int i = threadIdx.x; i < 1024; i += kT) {
      c.bucket[i] = 0;
      c.held[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kT) {
      const unsigned long long key = c.key[i];
      if (known < 64 && (key >> known) != prefix) continue;
      const unsigned d = (unsigned)(key >> shift) & 1023;
      atomicAdd(&c.held[d], 1u);
      if (by_mass) atomicAdd(&c.bucket[d], c.mass[i]);
    }
    __syncthreads();
    // this thread's digits, descending
    const int d0 = 1023 - 2 * threadIdx.x, d1 = d0 - 1;
    const unsigned n0 = c.held[d0], n1 = c.held[d1];
    const unsigned long long w0 = by_mass ? c.bucket[d0] : n0, w1 = by_mass ? c.bucket[d1] : n1;
    unsigned long long total;
    const unsigned long long at = before + block_scan_u64(w0 + w1, red, &total) - (w0 + w1);  // (all are read)
    if (at < limit && limit <= at + w0 + w1) {
      const bool second = limit > at + w0;
      c.bucket[0] = second ? d1 : d0;
      c.bucket[1] = at + (second ? w0 : 0);
      c.bucket[2] = second ? n1 : n0;
    }
    __syncthreads();
    prefix = prefix << (known - shift) | (c.bucket[0] & ((1ULL << (known - shift)) - 1));
    before = c.bucket[1];
    const bool one = c.bucket[2] == 1;
    known = shift;
    __syncthreads();
    if (one || known == 0) break;
    shift = max(shift - 10, 0);
  }
  for (int i = threadIdx.x; i < n; i += kT)
    if ((c.key[i] >> known) == prefix) c.bucket[0] = c.key[i];
  __syncthreads();
  return c.bucket[0];
}

// Of the keys from `last` on.
__device__ __forceinline__ unsigned long long total_mass(const Candidates &c, int n, unsigned long long last,
                                                         unsigned long long *red) {
  unsigned long long sum = 0, total;
  for (int i = threadIdx.x; i < n; i += kT) sum += c.key[i] >= last ? c.mass[i] : 0;
  block_scan_u64(sum, red, &total);
  return total;
}

// The bucket (of 1,024, ~0: none) on which `target` of the listed weights (of keys
// from `last` on) falls, in c.bucket[1] what of it is left there.
template <class Of>
__device__ __forceinline__ unsigned pick_bucket(Candidates &c, int n, unsigned long long last, unsigned long long target,
                                                unsigned long long *red, Of of) {
  __syncthreads();  // the last buckets are read
  for (int i = threadIdx.x; i < 1024; i += kT) c.bucket[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kT) {
    const unsigned b = of((unsigned)key_index(c.key[i]));
    if (b != ~0u && c.key[i] >= last && c.mass[i] != 0) atomicAdd(&c.bucket[b], c.mass[i]);
  }
  __syncthreads();
  const unsigned long long w0 = c.bucket[2 * threadIdx.x], w1 = c.bucket[2 * threadIdx.x + 1];
  unsigned long long total;
  const unsigned long long at = block_scan_u64(w0 + w1, red, &total) - (w0 + w1);  // (every bucket is read)
  if (at <= target && target < at + w0 + w1) {
    const bool second = target >= at + w0;
    c.bucket[0] = 2 * threadIdx.x + (second ? 1 : 0);
    c.bucket[1] = target - at - (second ? w0 : 0);
  }
  __syncthreads();
  return (unsigned)c.bucket[0];
}

// Everything from a list of all tokens that may be kept. limit: top-p's, 0: to be
// worked out of the list's weights (which are then all, or all that top-k keeps).
__device__ __forceinline__ int draw_listed(const SampleArgs &a, const RowParams &r, int row, Candidates &c, int n,
                                           unsigned long long limit, const double *table,
                                           unsigned long long *red) {
  weigh_candidates(r, c, n, table);
  unsigned long long last = 0;  // the last kept key
  if (r.k > 0 && r.k < n) last = last_key(c, n, false, 0, r.k, red);
  if (r.p < 1.0) last = last_key(c, n, true, 0, limit != 0 ? limit : limit_of(r.p, total_mass(c, n, last, red)), red);
  if (r.least > 0.0) {
    bool kept;
    for (int i = threadIdx.x; i < n; i += kT) {
      key_weight(r, c.key[i], table, &kept);
      if (!kept) c.mass[i] = 0;
    }
    __syncthreads();
  }
  // the token in the order of the indices: its upper ten bits, then its lower ten
  unsigned long long target = target_of(a, row, total_mass(c, n, last, red));
  const unsigned above = pick_bucket(c, n, last, target, red, [](unsigned i) { return i >> 10; });
  target = c.bucket[1];
  return (int)(above << 10 | pick_bucket(c, n, last, target, red, [above](unsigned i) { return (i >> 10) == above ? i & 1023 : ~0u; }));
}

// The first position in [begin, end) whose value is m.
__device__ __forceinline__ int first_of(const float *x, int begin, int end, float m, unsigned long long *red) {
  unsigned long long found = ~0ULL;
  for (int i = begin + 4 * (int)threadIdx.x; i < end && found == ~0ULL; i += 4 * kT) {
    const f32x4 v = load4(x, i, end);
#pragma unroll
    for (int e = 3; e >= 0; e--)
      if (v[e] == m && i + e < end) found = i + e;
  }
  return (int)block_min_u64(found, red);
}

__device__ __forceinline__ void load_table(const SampleArgs &a, double *table) {
  if (threadIdx.x < 64) table[threadIdx.x] = a.table[threadIdx.x];
  __syncthreads();
}

// ---- short rows ---------------------------------------------------------------------

__global__ __launch_bounds__(kT) void sample_short_kernel(const SampleArgs a) {
  __shared__ Candidates c;
  __shared__ double table[64];
  __shared__ unsigned long long red[kT / 64];
  __shared__ float fred[kT / 64];
  __shared__ unsigned int listed;
  const int row = blockIdx.x;
  const float *x = a.x + (size_t)row * a.ld;
  load_table(a, table);
  if (threadIdx.x == 0) listed = 0;
  const f32x4 v = load4(x, 4 * threadIdx.x, a.n);
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < 4; e++) m = fmaxf(m, v[e]);
  m = block_max(m, fred);
  const RowParams r = row_params(a, row, m);
  int found = -1;
  if (m > -INFINITY) {
    if (r.greedy) {
      found = first_of(x, 0, a.n, m, red);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float t = exponent(r, v[e]);
        if (t < kCutoff) c.key[atomicAdd(&listed, 1u)] = key_of(v[e], 4 * threadIdx.x + e);
      }
      __syncthreads();
      found = draw_listed(a, r, row, c, (int)listed, 0, table, red);
    }
  }
  if (threadIdx.x == 0) a.index[row] = found;
}

// ---- long rows ----------------------------------------------------------------------

__global__ __launch_bounds__(kT) void sample_max_kernel(const SampleArgs a) {
  constexpr int kU = 4;
  __shared__ float red[kT / 64];
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const float *x = a.x + (size_t)row * a.ld;
  RowState &s = a.rows[row];
  const int begin = split * a.chunk, end = min(begin + a.chunk, a.n);
  float m = -INFINITY;
  for (int i = begin + 4 * (int)threadIdx.x; i < end; i += 4 * kT * kU) {
    f32x4 v[kU];
#pragma unroll
    for (int u = 0; u < kU; u++) v[u] = load4(x, min(i + 4 * kT * u, end), end);
#pragma unroll
    for (int u = 0; u < kU; u++) m = fmaxf(fmaxf(fmaxf(m, v[u].x), fmaxf(v[u].y, v[u].z)), v[u].w);
  }
  for (int i = split * kT + threadIdx.x; i < kBins; i += a.splits * kT) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  m = block_max(m, red);
  if (threadIdx.x == 0) {
    s.split_max[split] = m;
    if (split == 0) s.listed = 0;
  }
}

__device__ __forceinline__ float row_max(const RowState &s, int splits) {
  const int lane = threadIdx.x & 63;
  float m = lane < splits ? s.split_max[lane] : -INFINITY;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  return m;
}

// use(v, i) of the row's values v[0 .. 3] at i .. i + 3, i from begin + 4 thread on, all
// lanes of a wave together; four vectors requested at once.
template <class Use>
__device__ __forceinline__ void each4(const float *x, int begin, int end, Use use) {
  constexpr int kU = 4;
  const int lane = threadIdx.x & 63;
  for (int i = begin + 4 * (int)threadIdx.x; i - 4 * lane < end; i += 4 * kT * kU) {
    f32x4 v[kU];
#pragma unroll
    for (int u = 0; u < kU; u++) v[u] = load4(x, min(i + 4 * kT * u, end), end);
#pragma unroll
    for (int u = 0; u < kU; u++)
      if (i + 4 * kT * u - 4 * lane < end) use(v[u], i + 4 * kT * u);
  }
}

__global__ __launch_bounds__(kT) void sample_bins_kernel(const SampleArgs a) {
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned int count[kBins];
  __shared__ double table[64];
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const float *x = a.x + (size_t)row * a.ld;
  RowState &s = a.rows[row];
  const RowParams r = row_params(a, row, row_max(s, a.splits));
  if (r.m == -INFINITY || r.greedy || (r.k == 0 && r.p >= 1.0)) return;
  for (int i = threadIdx.x; i < kBins; i += kT) {
    mass[i] = 0;
    count[i] = 0;
  }
  load_table(a, table);
  const int begin = split * a.chunk, end = min(begin + a.chunk, a.n);
  const bool weighed = r.k == 0;  // (where top-k ends, the counts say)
  each4(x, begin, end, [&](f32x4 v, int) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float t = exponent(r, v[e]);
      if (!(t < kCutoff)) continue;
      if (!weighed) {
        atomicAdd(&count[bin_of(t)], 1u);
        continue;
      }
      bool kept;
      const unsigned long long w = weight(r, v[e], table, &kept);
      atomicAdd(&mass[bin_of(t)], w);
      atomicAdd(&count[bin_of(t)], 1u);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kT)
    if (count[i] != 0) {
      if (weighed) atomicAdd(&s.mass[i], mass[i]);
      atomicAdd(&s.count[i], count[i]);
    }
}

__global__ __launch_bounds__(kT) void sample_gather_kernel(const SampleArgs a) {
  constexpr int kPer = kBins / kT;
  __shared__ double table[64];
  __shared__ unsigned long long red[kT / 64];
  __shared__ unsigned long long found[4], list[kList];
  __shared__ unsigned int listed, listed_at;
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const float *x = a.x + (size_t)row * a.ld;
  RowState &s = a.rows[row];
  const RowParams r = row_params(a, row, row_max(s, a.splits));
  if (r.m == -INFINITY || r.greedy) return;
  if (threadIdx.x == 0) listed = 0;
  load_table(a, table);
  int mode = kAll, bin = kBins, k = 0;
  unsigned long long limit = 0, before_mass = 0;
  unsigned int before_count = 0;
  if (r.k > 0 || r.p < 1.0) {
    unsigned long long mass[kPer], masses = 0, counts = 0, total_masses, total_counts;
    unsigned int count[kPer];
    const int i0 = threadIdx.x * kPer;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
      mass[e] = s.mass[i0 + e];
      count[e] = s.count[i0 + e];
      masses += mass[e];
      counts += count[e];
    }
    unsigned long long m0 = block_scan_u64(masses, red, &total_masses) - masses;
    unsigned long long c0 = block_scan_u64(counts, red, &total_counts) - counts;
    // (fewer tokens than top-k have a weight: it ends with the last of them)
    k = r.k > 0 ? (int)min((unsigned long long)r.k, total_counts) : 0;
    if (k == 0) limit = limit_of(r.p, total_masses);
    {
#pragma unroll
      for (int e = 0; e < kPer; e++) {
        // the bin that the k-th token, or the last one within the limit, is in
        const bool here = k > 0 ? c0 < (unsigned)k && (unsigned)k <= c0 + count[e]
                                : m0 < limit && limit <= m0 + mass[e];
        if (here) {
          found[0] = i0 + e;
          found[1] = c0;
          found[2] = m0;
          found[3] = count[e];
        }
        c0 += count[e];
        m0 += mass[e];
      }
      __syncthreads();
      bin = (int)found[0];
      before_count = (unsigned)found[1];
      before_mass = found[2];
      const unsigned in_bin = (unsigned)found[3];
      mode = before_count + in_bin <= kList ? kListed
             : in_bin <= kList && !(k > 0 && r.p < 1.0) ? kBinned
                                                        : kDigits;
    }
  }
  if (split == 0 && threadIdx.x == 0) {
    s.mode = mode;
    s.bin = bin;
    s.before_count = before_count;
    s.before_mass = before_mass;
    s.limit = limit;
    s.k = k;
  }
  if (mode == kDigits) return;
  const int begin = split * a.chunk, end = min(begin + a.chunk, a.n);
  // below this value no token is in the bins up to `bin` (by the bins' own factor, which
  // temperatures below 2^-126 meet the limit of; half a bin is more than the roundings of
  // t could make of it): most of the row is passed over by it
  const float least = mode == kAll || (r.k == 0 && bin == kBins - 1)
                          ? -INFINITY
                          : (float)((double)r.m - (bin + 1.5) / (0.5 * kBinsPerUnit * (double)r.inv_2t));
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i0 = begin + wave * kRun; i0 < end; i0 += kT / 64 * kRun) {
    unsigned long long sum = 0;
    f32x4 vs[kRun / kSegment];
#pragma unroll
    for (int u = 0; u < kRun / kSegment; u++) vs[u] = load4(x, min(i0 + u * kSegment + 4 * lane, end), end);
#pragma unroll
    for (int u = 0; u < kRun / kSegment; u++) {
      const f32x4 v = vs[u];
      const float top = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
      if (__ballot(!(top < least)) == 0) continue;  // (an infinite temperature below infinity: NaN)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float t = exponent(r, v[e]);
        const int b = t < kCutoff ? bin_of(t) : kBins + 1;
        if (mode != kListed && b < bin) {
          bool kept;
          const unsigned long long w = weight(r, v[e], table, &kept);
          sum += kept ? w : 0;
        }
        // (the bins' counts say that the list holds them all)
        if (mode != kAll && (mode == kListed ? b <= bin : b == bin)) {
          const unsigned int at = atomicAdd(&listed, 1u);
          if (at < kList) list[at] = key_of(v[e], i0 + u * kSegment + 4 * lane + e);
        }
      }
    }
    if (mode != kListed) {
      sum = wave_scan_u64(sum);
      if (lane == 63) s.run_mass[i0 / kRun] = sum;
    }
  }
  if (mode != kAll) {
    __syncthreads();
    if (threadIdx.x == 0 && listed > 0) listed_at = atomicAdd(&s.listed, listed);
    __syncthreads();
    for (unsigned int i = threadIdx.x; i < min(listed, (unsigned)kList); i += kT)
      if (listed_at + i < kList) s.list[listed_at + i] = list[i];
  }
}

// ---- the draw of long rows ------------------------------------------------------------

struct DrawLds {
  union {
    Candidates c;
    unsigned long long segment[kMaxSegments];
    struct {
      unsigned long long amount[256], mass[256];
    } digits;
  };
  double table[64];
  unsigned long long red[kT / 64], run_mass[kMaxRuns], shared[4];
};

// A token is kept: by its bin (before `bin`), or its key (`last`: the last kept
// one's), and min_p. Its weight, or 0.
__device__ __forceinline__ unsigned long long kept_weight(const RowParams &r, float x, int i, int bin,
                                                          unsigned long long last, const double *table) {
  const float t = exponent(r, x);
  if (!(t < kCutoff)) return 0;
  if (!(bin_of(t) < bin) && key_of(x, i) < last) return 0;
  bool kept;
  const unsigned long long w = weight(r, x, table, &kept);
  return kept ? w : 0;
}

// The token of [begin, end) on which `target` of the kept weights from `begin` on
// falls; with pick false only their sum. A segment of 256 tokens per wave and
// step, its sum in LDS.
__device__ __forceinline__ unsigned long long segment_sums(const RowParams &r, const float *x, int begin, int end,
                                                           int bin, unsigned long long last, DrawLds &lds) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int segments = (end - begin + kSegment - 1) / kSegment;
  __syncthreads();
  for (int g = wave; g < segments; g += kT / 64) {
    const int i = begin + g * kSegment + 4 * lane;
    const f32x4 v = load4(x, min(i, end), end);
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) sum += kept_weight(r, v[e], i + e, bin, last, lds.table);
    sum = wave_scan_u64(sum);
    if (lane == 63) lds.segment[g] = sum;
  }
  __syncthreads();
  unsigned long long sum = 0, total;
  for (int g = threadIdx.x; g < segments; g += kT) sum += lds.segment[g];
  block_scan_u64(sum, lds.red, &total);
  return total;
}

__device__ __forceinline__ int pick(const RowParams &r, const float *x, int begin, int end, int bin,
                                    unsigned long long last, unsigned long long target, DrawLds &lds) {
  const int segments = (end - begin + kSegment - 1) / kSegment, lane = threadIdx.x & 63;
  // the segment: each thread looks through a run of them
  const int per = (segments + kT - 1) / kT, g0 = threadIdx.x * per;
  unsigned long long sum = 0, total;
  for (int g = g0; g < min(g0 + per, segments); g++) sum += lds.segment[g];
  unsigned long long at = block_scan_u64(sum, lds.red, &total) - sum;
  for (int g = g0; g < min(g0 + per, segments); g++) {
    const unsigned long long w = lds.segment[g];
    if (at <= target && target < at + w) {
      lds.shared[0] = g;
      lds.shared[1] = at;
    }
    at += w;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int i = begin + (int)lds.shared[0] * kSegment + 4 * lane;
    const f32x4 v = load4(x, min(i, end), end);
    unsigned long long w[4], mine = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      w[e] = kept_weight(r, v[e], i + e, bin, last, lds.table);
      mine += w[e];
    }
    unsigned long long to = lds.shared[1] + wave_scan_u64(mine) - mine;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (to <= target && target < to + w[e]) lds.shared[2] = i + e;
      to += w[e];
    }
  }
  __syncthreads();
  return (int)lds.shared[2];
}

// The token that u falls on, from the runs' weights.
__device__ __forceinline__ int pick_in_run(const SampleArgs &a, const RowParams &r, const float *x, int row, int bin,
                                           unsigned long long last, DrawLds &lds) {
  constexpr int kPer = kMaxRuns / kT;
  static_assert(kMaxRuns % kT == 0 && kRun <= 4 * kT, "some runs per thread, then four tokens");
  unsigned long long total, sum = 0;
  const int g0 = kPer * (int)threadIdx.x;
#pragma unroll
  for (int e = 0; e < kPer; e++) sum += lds.run_mass[g0 + e];
  unsigned long long at = block_scan_u64(sum, lds.red, &total) - sum;
  const unsigned long long target = target_of(a, row, total);
#pragma unroll
  for (int e = 0; e < kPer; e++) {
    const unsigned long long w = lds.run_mass[g0 + e];
    if (at <= target && target < at + w) {
      lds.shared[0] = g0 + e;
      lds.shared[1] = at;
    }
    at += w;
  }
  __syncthreads();
  const int i = (int)lds.shared[0] * kRun + 4 * (int)threadIdx.x;
  const int end = min((int)(lds.shared[0] + 1) * kRun, a.n);
  const f32x4 v = load4(x, min(i, end), end);
  unsigned long long w[4], mine = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    w[e] = kept_weight(r, v[e], i + e, bin, last, lds.table);
    mine += w[e];
  }
  at = lds.shared[1] + block_scan_u64(mine, lds.red, &sum) - mine;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (at <= target && target < at + w[e]) lds.shared[2] = i + e;
    at += w[e];
  }
  __syncthreads();
  return (int)lds.shared[2];
}

// The first key, descending, at which the tokens' counts (by_mass false) or
// weights up to it and with it reach `limit`, 8 bits of the key at a time;
// *mass: the weights up to it and with it.
__device__ unsigned long long key_at(const RowParams &r, const float *x, int n, bool by_mass,
                                     unsigned long long limit, DrawLds &lds, unsigned long long *mass) {
  unsigned long long prefix = 0, before = 0, before_mass = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kT) lds.digits.amount[i] = lds.digits.mass[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kT) {
      const float v = x[i];
      const float t = exponent(r, v);
      const unsigned long long key = key_of(v, i);
      if (!(t < kCutoff) || (shift < 56 && (key >> (shift + 8)) != prefix)) continue;
      bool kept;
      const unsigned long long w = weight(r, v, lds.table, &kept);
      atomicAdd(&lds.digits.mass[(key >> shift) & 255], w);
      atomicAdd(&lds.digits.amount[(key >> shift) & 255], by_mass ? w : 1ULL);
    }
    __syncthreads();
    // threads 0 .. 255 hold the digits from 255 down
    const int d = 255 - (int)threadIdx.x;
    const unsigned long long amount = d >= 0 ? lds.digits.amount[d] : 0, w = d >= 0 ? lds.digits.mass[d] : 0;
    unsigned long long total;
    const unsigned long long c = before + block_scan_u64(amount, lds.red, &total);
    const unsigned long long m = before_mass + block_scan_u64(w, lds.red, &total);
    if (d >= 0 && c - amount < limit && limit <= c) {
      lds.shared[0] = (prefix << 8) | (unsigned)d;
      lds.shared[1] = c - amount;
      lds.shared[2] = m - w;
      lds.shared[3] = m;
    }
    __syncthreads();
    prefix = lds.shared[0];
    before = lds.shared[1];
    before_mass = lds.shared[2];
    *mass = lds.shared[3];
  }
  return prefix;
}

__global__ __launch_bounds__(kT) void sample_draw_kernel(const SampleArgs a) {
  __shared__ DrawLds lds;
  const int row = blockIdx.x;
  const float *x = a.x + (size_t)row * a.ld;
  const RowState &s = a.rows[row];
  const RowParams r = row_params(a, row, row_max(s, a.splits));
  load_table(a, lds.table);
  int found = -1;
  if (r.m > -INFINITY && r.greedy) {
    int split = 0;
    while (split < a.splits - 1 && s.split_max[split] != r.m) split++;
    found = first_of(x, split * a.chunk, min((split + 1) * a.chunk, a.n), r.m, lds.red);
  } else if (r.m > -INFINITY) {
    const int listed = (int)min(s.listed, (unsigned)kList), mode = s.mode;
    int bin = s.bin;
    unsigned long long last = ~0ULL;
    if (mode == kListed || mode == kBinned) {
      for (int i = threadIdx.x; i < listed; i += kT) lds.c.key[i] = s.list[i];
      __syncthreads();
    }
    if (mode == kListed) {
      found = draw_listed(a, r, row, lds.c, listed, s.limit, lds.table, lds.red);
    } else if (mode == kDigits) {
      unsigned long long mass = 0, limit = s.limit;
      last = 0;
      bin = 0;
      if (s.k > 0) {
        last = key_at(r, x, a.n, false, (unsigned long long)s.k, lds, &mass);
        limit = r.p < 1.0 ? limit_of(r.p, mass) : 0;
      }
      if (limit > 0) last = key_at(r, x, a.n, true, limit, lds, &mass);
      const unsigned long long total = segment_sums(r, x, 0, a.n, bin, last, lds);
      found = pick(r, x, 0, a.n, bin, last, target_of(a, row, total), lds);
    } else {
      for (int i = threadIdx.x; i < kMaxRuns; i += kT) lds.run_mass[i] = i * kRun < a.n ? s.run_mass[i] : 0;
      __syncthreads();
      if (mode == kBinned) {
        weigh_candidates(r, lds.c, listed, lds.table);
        last = s.k > 0 ? last_key(lds.c, listed, false, s.before_count, s.k, lds.red)
                       : last_key(lds.c, listed, true, s.before_mass, s.limit, lds.red);
        for (int i = threadIdx.x; i < listed; i += kT) {
          bool above;
          const unsigned long long key = lds.c.key[i], w = key_weight(r, key, lds.table, &above);
          if (above && key >= last) atomicAdd(&lds.run_mass[key_index(key) / kRun], w);
        }
        __syncthreads();
      }
      found = pick_in_run(a, r, x, row, bin, last, lds);
    }
  }
  if (threadIdx.x == 0) a.index[row] = found;
}

// Splits of a row: about 1,024 workgroups in all, of at least 2,048 logits each.
void sample_split(int rows, int n, int *splits, int *chunk) {
  const int unit = 4 * kT;
  const long long most = std::min<long long>(kMaxSplits, (n + unit - 1) / unit);
  const long long want = std::max(1LL, std::min(most, (long long)(1024 + rows - 1) / rows));
  *chunk = (int)((n + want * unit - 1) / (want * unit)) * unit;
  *splits = (n + *chunk - 1) / *chunk;
}

size_t workspace_of(int rows, int n) { return n <= kList ? 16 : (size_t)rows * sizeof(RowState); }

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_sample_workspace(int rows, int n, size_t *bytes) {
  if (!bytes) return fail(SH_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (const char *wrong = check_sample_sizes(rows, n, n)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  *bytes = workspace_of(rows, n);
  return SH_OK;
}

SH_API int sh_sample_f32(sh_ctx *ctx, const float *x, int rows, int n, int ld, const float *temperature,
                         const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                         int32_t *index, void *workspace, size_t workspace_bytes) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (const char *wrong = check_sample_sizes(rows, n, ld)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (rows == 0) return SH_OK;
  const size_t per_row = (size_t)rows * 4, need = workspace_of(rows, n);
  if ((rc = check_range(ctx, x, ((size_t)(rows - 1) * ld + n) * 4, "x")) ||
      (temperature && (rc = check_range(ctx, temperature, per_row, "temperature"))) ||
      (top_k && (rc = check_range(ctx, top_k, per_row, "top_k"))) ||
      (top_p && (rc = check_range(ctx, top_p, per_row, "top_p"))) ||
      (min_p && (rc = check_range(ctx, min_p, per_row, "min_p"))) || (rc = check_range(ctx, u, per_row, "u")) ||
      (rc = check_range(ctx, index, per_row, "index")))
    return rc;
  if (workspace_bytes < need)
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer has %zu bytes, %zu are needed", workspace_bytes, need);
  if ((rc = check_range(ctx, workspace, need, "workspace"))) return rc;
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer must be 16-byte aligned");
  // (a row's values by scalar loads, which leave the last two bits of an address out; NULL is aligned)
  if ((reinterpret_cast<uintptr_t>(temperature) | reinterpret_cast<uintptr_t>(top_k) | reinterpret_cast<uintptr_t>(top_p) |
       reinterpret_cast<uintptr_t>(min_p) | reinterpret_cast<uintptr_t>(u)) & 3)
    return fail(SH_ERR_INVALID_ARGUMENT, "temperature, top_k, top_p, min_p and u must be 4-byte aligned");
  // what a call writes (rows that the list holds use no work buffer) lies over nothing that it reads
  const size_t x_bytes = ((size_t)(rows - 1) * ld + n) * 4;
  if (n > kList && ranges_overlap(workspace, need, x, x_bytes))
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer overlaps x");
  const auto over_parameters = [&](const void *p, size_t bytes) {
    for (const void *of : {(const void *)temperature, (const void *)top_k, (const void *)top_p, (const void *)min_p, (const void *)u})
      if (of && ranges_overlap(p, bytes, of, per_row)) return true;
    return false;
  };
  if (n > kList && (over_parameters(workspace, need) || ranges_overlap(workspace, need, index, per_row)))
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer overlaps index, u or a row's parameters");
  if (ranges_overlap(index, per_row, x, x_bytes) || over_parameters(index, per_row))
    return fail(SH_ERR_INVALID_ARGUMENT, "index overlaps x, u or a row's parameters");
  SampleArgs a;
  a.x = x;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.u = u;
  a.index = index;
  a.rows = static_cast<RowState *>(workspace);
  a.n = n;
  a.ld = ld;
  for (int j = 0; j < 64; j++) a.table[j] = std::exp2(-j / 64.0);
  const hipStream_t st = stream_of(ctx);
  if (n <= kList) {
    a.splits = 1;
    a.chunk = n;
    sample_short_kernel<<<rows, kT, 0, st>>>(a);
  } else {
    sample_split(rows, n, &a.splits, &a.chunk);
    const unsigned grid = (unsigned)rows * (unsigned)a.splits;
    sample_max_kernel<<<grid, kT, 0, st>>>(a);
    sample_bins_kernel<<<grid, kT, 0, st>>>(a);
    sample_gather_kernel<<<grid, kT, 0, st>>>(a);
    sample_draw_kernel<<<rows, kT, 0, st>>>(a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "sample");
}

}  // extern "C"
