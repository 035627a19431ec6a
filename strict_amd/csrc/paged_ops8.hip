// What goes into a KV cache in pages of 8-bit values and comes out of it: the head norms
// and RoPE of new tokens with their k and v quantised into pages, and rows read back (the
// pages' layout: paged.h).
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.h"
#include "paged.h"
#include "paged_device.h"

namespace sh {
namespace {

constexpr int kT = 256;

struct NormRope8Args {
  const uint16_t *qkv;
  const float *q_gain, *k_gain;
  uint16_t *q;
  uint8_t *pages;
  const int *table, *lengths, *starts;
  size_t page_bytes;
  int tokens, batch, max_pages, num_pages, page_shift, heads, kv_heads, ld, chunks;
  float eps;
  double freq[64];  // theta^(-2i / d)
};

// A token's row of the call: its position, and the page of it (-1: none).
struct TokenPlace {
  bool there;  // of a sequence
  int pos, page;
};
__device__ __forceinline__ TokenPlace token_place(const int *starts, const int *lengths, const int *table, int batch,
                                                  int tokens, int max_pages, int num_pages, int page_shift, int row) {
  TokenPlace p = {false, 0, -1};
  const int b = find_seq(starts, batch, row);
  if (b < 0 || b >= batch) return p;
  const PagedSeq s = paged_seq(starts[b], starts[b + 1], lengths[b], tokens, max_pages << page_shift);
  p.there = true;
  p.pos = s.len - s.n + (row - s.row0);
  if (p.pos >= 0 && p.pos < s.len) p.page = paged_page(table[(size_t)b * max_pages + (p.pos >> page_shift)], num_pages);
  return p;
}

// The largest value that E4M3 times a power of two and the 16-bit type both hold: 1.875
// times the type's largest power of two.
template <class T>
constexpr float kLargest8 = T::kIsF16 ? 0x1.ep15f : 0x1.ep127f;

// A magnitude in 64 bits as a key that orders as it does: its upper word, and whether there
// is anything in the lower one. 20 bits behind the point and that bit are what rounding to
// E4M3's 3, half way to even, can depend on.
__device__ __forceinline__ uint32_t size_key(double y) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, y);
  return ((uint32_t)(bits >> 32) << 1) | min((uint32_t)bits, 1u);
}
// The exponent of the scale of a row whose largest key is `most`: 448 = 1.75 * 2^8.
__device__ __forceinline__ int row_exponent(uint32_t most) {
  return max((int)(most >> 21) - 1023 - 8 + ((most & 0x1fffff) > 0x180000 ? 1 : 0), -127);
}
// Its value times 2^-exponent in fp32, the key's last bit in the fraction. (What is far below
// E4M3's smallest comes to 0.)
__device__ __forceinline__ float key_value(double y, uint32_t key, int exponent) {
  const uint32_t sign = (uint32_t)(__builtin_bit_cast(uint64_t, y) >> 32) & 0x80000000u;
  return __builtin_bit_cast(float, ((uint32_t)max((int)(key - ((uint32_t)(1023 - 127 + exponent) << 21)), 0) << 2) | sign);
}

// 2^e, e of -126 .. 127.
__device__ __forceinline__ float exponent_value(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }

// To fp32 with the last bit set where something was cut off: rounding that to fewer bits
// by at least two gives what rounding the fp64 value at once would.
__device__ __forceinline__ float to_odd(double x) {
  const float f = __double2float_rz(x);
  return (double)f != x && f == f ? __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f) | 1u) : f;
}

typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  s16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, 1.0f, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, 1.0f, true);
  return __builtin_bit_cast(uint32_t, r);
}

// Of kLanes (4 or 8) lanes that follow each other: by lane moves, a fraction of the time of
// LDS permutes.
template <int kCtrl>
__device__ __forceinline__ uint32_t lane_move(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, false);
}
template <int kCtrl>
__device__ __forceinline__ float lane_move(float v) {
  return __builtin_bit_cast(float, lane_move<kCtrl>(__builtin_bit_cast(uint32_t, v)));
}
template <int kCtrl>
__device__ __forceinline__ double lane_move(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, ((uint64_t)lane_move<kCtrl>((uint32_t)(u >> 32)) << 32) | lane_move<kCtrl>((uint32_t)u));
}
template <int kLanes, class V, class Op>
__device__ __forceinline__ V over_lanes(V v, Op op) {
  v = op(v, lane_move<0xb1>(v));                              // lane ^ 1
  v = op(v, lane_move<0x4e>(v));                              // lane ^ 2
  if constexpr (kLanes == 8) v = op(v, lane_move<0x141>(v));  // 7 - lane: the other four
  return v;
}

// A wave takes kSteps * kHeadsAt heads of one token: q heads, then k, then v. A head is
// d / 16 lanes wide, 8 values of its first half and the 8 that rotate with them in each
// lane, all loads requested at once. q is worked out as for the 16-bit cache, bit for bit. k
// is normalised and rotated in fp64 (which has fp32's rate here) so that its bytes do not
// depend on the order of sums: in fp32 one value in 10^6 comes out a step of E4M3, 6 % of
// it, off. (Quantised in fp64 too, v as well, and with sums by LDS permutes:
// 41 us for 9,312 tokens of 16 and 8 heads of 128 and not 28.5, 8.2 us for 3 and not 3.5.)
// Bound by the bytes: those 9,312 are 172 MB, 6.0 TB/s. (Stores of pages that the caches
// need not keep take as long, and reading the rows back 14.6 us and not 13.)
template <class T, int kD, int kSteps>
__global__ __launch_bounds__(kT) void norm_rope8_kernel(const NormRope8Args a) {
  constexpr int kLanes = kD / 16, kHeadsAt = 64 / kLanes, kHalf = kD / 2;
  __shared__ double2 factors[kT / 64][kHalf];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long unit = (long long)blockIdx.x * (kT / 64) + wave;
  if (unit >= (long long)a.tokens * a.chunks) return;
  const int row = __builtin_amdgcn_readfirstlane((int)(unit / a.chunks));
  const int h0 = __builtin_amdgcn_readfirstlane((int)(unit % a.chunks)) * kHeadsAt * kSteps;
  const int all = a.heads + 2 * a.kv_heads, part = lane % kLanes, sub = lane / kLanes;
  const uint16_t *x = a.qkv + (size_t)row * a.ld + part * 8;
  u32x4 lo[kSteps], hi[kSteps];
#pragma unroll
  for (int u = 0; u < kSteps; u++) {
    const int h = min(h0 + u * kHeadsAt + sub, all - 1);
    lo[u] = *reinterpret_cast<const u32x4 *>(x + (size_t)h * kD);
    hi[u] = *reinterpret_cast<const u32x4 *>(x + (size_t)h * kD + kHalf);
  }
  const TokenPlace p = token_place(a.starts, a.lengths, a.table, a.batch, a.tokens, a.max_pages, a.num_pages,
                                   a.page_shift, row);
  if (!p.there) return;
  if (lane < kHalf) {
    double c, sn;
    cos_sin64((double)p.pos * a.freq[lane], &c, &sn);
    factors[wave][lane] = make_double2(c, sn);
  }
  __builtin_amdgcn_wave_barrier();
  const int in_page = p.pos & ((1 << a.page_shift) - 1);
  const size_t v_at = ((size_t)a.kv_heads << a.page_shift) * kD;  // of a page
  uint8_t *page = a.pages + (size_t)max(p.page, 0) * a.page_bytes;
#pragma unroll
  for (int u = 0; u < kSteps; u++) {
    const int h = h0 + u * kHeadsAt + sub;
    float x1[8], x2[8];
    unpack8<T>(lo[u], x1);
    unpack8<T>(hi[u], x2);
    if (h < a.heads) {
      head_norm_rope<kD>(x1, x2, a.q_gain + part * 8, a.eps, [&](int e) {
        const double2 f = factors[wave][part * 8 + e];
        return make_float2((float)f.x, (float)f.y);
      });
      uint16_t *to = a.q + ((size_t)row * a.heads + h) * kD + part * 8;
      __builtin_nontemporal_store(pack8<T>(x1), reinterpret_cast<u32x4 *>(to));
      __builtin_nontemporal_store(pack8<T>(x2), reinterpret_cast<u32x4 *>(to + kHalf));
      continue;
    }
    if (h >= all || p.page < 0) continue;
    const bool is_k = h < a.heads + a.kv_heads;
    const int kv_head = h - a.heads - (is_k ? 0 : a.kv_heads);
    int exponent = 0;
    bool plain;  // nothing beyond the largest, or not finite, in the lane: x1, x2 are scaled
    if (is_k) {
      double y1[8], y2[8], ss = 0.0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y1[e] = x1[e];
        y2[e] = x2[e];
        ss = fma(y1[e], y1[e], fma(y2[e], y2[e], ss));
      }
      ss = over_lanes<kLanes>(ss, [](double m, double n) { return m + n; });
      const double inv = 1.0 / sqrt(ss * (1.0 / kD) + a.eps);
      const float *gain = a.k_gain + part * 8;
      uint32_t key1[8], key2[8], most = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const double2 f = factors[wave][part * 8 + e];
        const double z1 = y1[e] * (inv * gain[e]), z2 = y2[e] * (inv * gain[e + kHalf]);
        y1[e] = fma(z1, f.x, -(z2 * f.y));
        y2[e] = fma(z2, f.x, z1 * f.y);
        key1[e] = size_key(y1[e]);
        key2[e] = size_key(y2[e]);
        most = max(most, max(key1[e], key2[e]));
      }
      most = over_lanes<kLanes>(most, [](uint32_t m, uint32_t n) { return max(m, n); });
      plain = most <= size_key((double)kLargest8<T>);
      if (plain) {
        exponent = row_exponent(most);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x1[e] = key_value(y1[e], key1[e], exponent);
          x2[e] = key_value(y2[e], key2[e], exponent);
        }
      } else {  // (to fp32 for what follows: the last bit stands for all that is cut off)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x1[e] = to_odd(y1[e]);
          x2[e] = to_odd(y2[e]);
        }
      }
    } else {
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) most = fmaxf(most, fmaxf(__builtin_fabsf(x1[e]), __builtin_fabsf(x2[e])));
      most = over_lanes<kLanes>(most, [](float m, float n) { return fmaxf(m, n); });
      plain = most <= kLargest8<T>;
      if (plain) {
        exponent = row_exponent(size_key((double)most));
        const float to_row = exponent_value(-exponent);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          x1[e] *= to_row;
          x2[e] *= to_row;
        }
      }
    }
    if (!plain) {  // infinities become NaN, which the maximum passes over and the format keeps
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        for (float *y : {&x1[e], &x2[e]}) {
          const float size = __builtin_fabsf(*y);
          *y = size == INFINITY ? NAN : size > kLargest8<T> ? copysignf(kLargest8<T>, *y) : *y;
          most = fmaxf(most, __builtin_fabsf(*y));
        }
      }
      most = over_lanes<kLanes>(most, [](float m, float n) { return fmaxf(m, n); });
      exponent = row_exponent(size_key((double)most));
      const float to_row = exponent_value(-exponent);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x1[e] *= to_row;
        x2[e] *= to_row;
      }
    }
    const size_t at = ((size_t)kv_head << a.page_shift) + in_page;
    uint8_t *to = page + (is_k ? 0 : v_at) + at * kD + part * 8;
    const u32x2 b1 = {to_e4m3(x1[0], x1[1], x1[2], x1[3]), to_e4m3(x1[4], x1[5], x1[6], x1[7])};
    const u32x2 b2 = {to_e4m3(x2[0], x2[1], x2[2], x2[3]), to_e4m3(x2[4], x2[5], x2[6], x2[7])};
    *reinterpret_cast<u32x2 *>(to) = b1;
    *reinterpret_cast<u32x2 *>(to + kHalf) = b2;
    if (part == 0) page[2 * v_at + (is_k ? 0 : (size_t)a.kv_heads << a.page_shift) + at] = (uint8_t)(exponent + 127);
  }
}

template <class T, int kD>
void launch_norm_rope8(hipStream_t st, NormRope8Args &a) {
  constexpr int kHeadsAt = 64 / (kD / 16);
  const int all = a.heads + 2 * a.kv_heads;
  const auto grid = [&](int steps) {
    a.chunks = (all + steps * kHeadsAt - 1) / (steps * kHeadsAt);
    return (unsigned)(((long long)a.tokens * a.chunks + kT / 64 - 1) / (kT / 64));
  };
  // of few tokens a step each, side by side
  if ((long long)a.tokens * all <= 2048LL * kHeadsAt) {
    const unsigned blocks = grid(1);
    norm_rope8_kernel<T, kD, 1><<<blocks, kT, 0, st>>>(a);
  } else {
    const unsigned blocks = grid(4);
    norm_rope8_kernel<T, kD, 4><<<blocks, kT, 0, st>>>(a);
  }
}

template <class T>
int norm_rope8(sh_ctx *ctx, const sh_paged_kv8 *kv, const uint16_t *qkv, const float *q_gain,
               const float *k_gain, uint16_t *q, int tokens, int heads, int ld, float eps, float theta) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (!kv) return fail(SH_ERR_INVALID_ARGUMENT, "the paged cache is NULL");
  const sh_paged_kv index = paged8_index(kv);
  if (const char *wrong = check_paged_sizes(&index, tokens, heads)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  const int d = kv->head_dim;
  if (!paged_dim_built(d)) return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", d);
  if (!(eps >= 0.0f)) return fail(SH_ERR_INVALID_ARGUMENT, "eps must be >= 0");
  if (const char *wrong = check_rope_theta(&index, tokens, theta)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  const long long width = ((long long)heads + 2LL * kv->kv_heads) * d;
  if (ld < width || ld % 8 != 0)
    return fail(SH_ERR_INVALID_ARGUMENT, "ld %d must be a multiple of 8 and at least %lld", ld, width);
  if (tokens == 0 || kv->batch == 0) return SH_OK;
  const size_t in_bytes = ((size_t)(tokens - 1) * ld + (size_t)width) * 2, q_bytes = (size_t)tokens * heads * d * 2;
  const size_t gain_bytes = (size_t)d * 4, pool = paged8_pool_bytes(kv);
  if ((rc = check_paged8_pointers(ctx, kv)) || (rc = check_range(ctx, qkv, in_bytes, "qkv")) ||
      (rc = check_range(ctx, q_gain, gain_bytes, "q_gain")) || (rc = check_range(ctx, k_gain, gain_bytes, "k_gain")) ||
      (rc = check_range(ctx, q, q_bytes, "q")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "qkv and q must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(q_gain) | reinterpret_cast<uintptr_t>(k_gain)) & 3)
    return fail(SH_ERR_INVALID_ARGUMENT, "the gains must be 4-byte aligned");
  if (ranges_overlap(qkv, in_bytes, q, q_bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "q overlaps qkv");
  if (ranges_overlap(kv->pages, pool, q, q_bytes) || ranges_overlap(kv->pages, pool, qkv, in_bytes))
    return fail(SH_ERR_INVALID_ARGUMENT, "the cache overlaps q or qkv");
  const auto over_inputs = [&](const void *p, size_t bytes) {
    return overlaps_index(&index, p, bytes) || ranges_overlap(p, bytes, q_gain, gain_bytes) ||
           ranges_overlap(p, bytes, k_gain, gain_bytes);
  };
  if (over_inputs(q, q_bytes) || over_inputs(kv->pages, pool))
    return fail(SH_ERR_INVALID_ARGUMENT, "q or the cache overlaps the page table, lengths, starts or gains");
  NormRope8Args a;
  a.qkv = qkv;
  a.q_gain = q_gain;
  a.k_gain = k_gain;
  a.q = q;
  a.pages = kv->pages;
  a.table = kv->page_table;
  a.lengths = kv->lengths;
  a.starts = kv->starts;
  a.page_bytes = paged8_page_bytes(kv);
  a.tokens = tokens;
  a.batch = kv->batch;
  a.max_pages = kv->max_pages;
  a.num_pages = kv->num_pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  a.heads = heads;
  a.kv_heads = kv->kv_heads;
  a.ld = ld;
  a.eps = eps;
  rope_frequencies(theta, d, a.freq);
  if (d == 64)
    launch_norm_rope8<T, 64>(stream_of(ctx), a);
  else
    launch_norm_rope8<T, 128>(stream_of(ctx), a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "qk_norm_rope_paged8");
}

// ---- rows read back ---------------------------------------------------------------------

struct Read8Args {
  const uint8_t *pages;
  uint16_t *k, *v;
  const int *table, *lengths, *starts;
  size_t page_bytes;
  int tokens, batch, max_pages, num_pages, page_shift, kv_heads, chunks;
};

// A wave takes 4 * kRowsAt of a token's 2 kv_heads rows, k first; a row is d / 16 lanes
// wide. 9,312 tokens of 8 heads of 128 (57 MB) take 13 us, 4.4 TB/s: of fewer rows than a wave
// has places (there 16 of 32) the others' loads repeat the last row.
template <class T, int kD>
__global__ __launch_bounds__(kT) void read8_kernel(const Read8Args a) {
  constexpr int kLanes = kD / 16, kRowsAt = 64 / kLanes, kSteps = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long unit = (long long)blockIdx.x * (kT / 64) + wave;
  if (unit >= (long long)a.tokens * a.chunks) return;
  const int row = __builtin_amdgcn_readfirstlane((int)(unit / a.chunks));
  const int r0 = __builtin_amdgcn_readfirstlane((int)(unit % a.chunks)) * kRowsAt * kSteps;
  const TokenPlace p = token_place(a.starts, a.lengths, a.table, a.batch, a.tokens, a.max_pages, a.num_pages,
                                   a.page_shift, row);
  if (!p.there || p.page < 0) return;
  const int rows = 2 * a.kv_heads, part = lane % kLanes, in_page = p.pos & ((1 << a.page_shift) - 1);
  const uint8_t *page = a.pages + (size_t)p.page * a.page_bytes;
  const size_t scales = ((size_t)rows << a.page_shift) * kD;
  u32x4 x[kSteps];
  uint32_t scale[kSteps];
#pragma unroll
  for (int u = 0; u < kSteps; u++) {
    const int r = min(r0 + u * kRowsAt + lane / kLanes, rows - 1);
    const size_t at = ((size_t)r << a.page_shift) + in_page;  // (the heads of v follow those of k)
    x[u] = *reinterpret_cast<const u32x4 *>(page + at * kD + part * 16);
    scale[u] = page[scales + at];
  }
#pragma unroll
  for (int u = 0; u < kSteps; u++) {
    const int r = r0 + u * kRowsAt + lane / kLanes;
    if (r >= rows) continue;
    const float s = e8m0_scale(scale[u]);
    uint16_t *to = (r < a.kv_heads ? a.k + ((size_t)row * a.kv_heads + r) * kD
                                   : a.v + ((size_t)row * a.kv_heads + (r - a.kv_heads)) * kD) +
                   part * 16;
    __builtin_nontemporal_store(from_e4m3<T>(x[u].x, x[u].y, s), reinterpret_cast<u32x4 *>(to));
    __builtin_nontemporal_store(from_e4m3<T>(x[u].z, x[u].w, s), reinterpret_cast<u32x4 *>(to + 8));
  }
}

template <class T>
int read8(sh_ctx *ctx, const sh_paged_kv8 *kv, uint16_t *k, uint16_t *v, int tokens) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (!kv) return fail(SH_ERR_INVALID_ARGUMENT, "the paged cache is NULL");
  const sh_paged_kv index = paged8_index(kv);
  if (const char *wrong = check_paged_sizes(&index, tokens, kv->kv_heads))
    return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  const int d = kv->head_dim;
  if (!paged_dim_built(d)) return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", d);
  if (tokens == 0 || kv->batch == 0) return SH_OK;
  const size_t bytes = (size_t)tokens * kv->kv_heads * d * 2, pool = paged8_pool_bytes(kv);
  if ((rc = check_paged8_pointers(ctx, kv)) || (rc = check_range(ctx, k, bytes, "k")) ||
      (rc = check_range(ctx, v, bytes, "v")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "k and v must be 16-byte aligned");
  if (ranges_overlap(k, bytes, v, bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "k overlaps v");
  for (const uint16_t *p : {k, v})
    if (ranges_overlap(p, bytes, kv->pages, pool) || overlaps_index(&index, p, bytes))
      return fail(SH_ERR_INVALID_ARGUMENT, "k or v overlaps the cache, the page table, lengths or starts");
  Read8Args a;
  a.pages = kv->pages;
  a.k = k;
  a.v = v;
  a.table = kv->page_table;
  a.lengths = kv->lengths;
  a.starts = kv->starts;
  a.page_bytes = paged8_page_bytes(kv);
  a.tokens = tokens;
  a.batch = kv->batch;
  a.max_pages = kv->max_pages;
  a.num_pages = kv->num_pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  a.kv_heads = kv->kv_heads;
  const int per_unit = 4 * (64 / (d / 16));
  a.chunks = (2 * kv->kv_heads + per_unit - 1) / per_unit;
  const long long units = (long long)tokens * a.chunks;
  const unsigned grid = (unsigned)((units + kT / 64 - 1) / (kT / 64));
  if (d == 64)
    read8_kernel<T, 64><<<grid, kT, 0, stream_of(ctx)>>>(a);
  else
    read8_kernel<T, 128><<<grid, kT, 0, stream_of(ctx)>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "paged8_read");
}

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_paged8_page_bytes(const sh_paged_kv8 *kv, size_t *bytes) {
  if (!kv) return fail(SH_ERR_INVALID_ARGUMENT, "the paged cache is NULL");
  if (!bytes) return fail(SH_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const sh_paged_kv index = paged8_index(kv);
  if (const char *wrong = check_paged_sizes(&index, 0, kv->kv_heads)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (!paged_dim_built(kv->head_dim))
    return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", kv->head_dim);
  *bytes = paged8_page_bytes(kv);
  return SH_OK;
}

SH_API int sh_qk_norm_rope_paged8_f16(sh_ctx *ctx, const sh_paged_kv8 *kv, const uint16_t *qkv,
                                      const float *q_gain, const float *k_gain, uint16_t *q, int tokens,
                                      int heads, int ld, float eps, float theta) {
  return norm_rope8<PagedF16>(ctx, kv, qkv, q_gain, k_gain, q, tokens, heads, ld, eps, theta);
}

SH_API int sh_qk_norm_rope_paged8_bf16(sh_ctx *ctx, const sh_paged_kv8 *kv, const uint16_t *qkv,
                                       const float *q_gain, const float *k_gain, uint16_t *q, int tokens,
                                       int heads, int ld, float eps, float theta) {
  return norm_rope8<PagedBf16>(ctx, kv, qkv, q_gain, k_gain, q, tokens, heads, ld, eps, theta);
}

SH_API int sh_paged8_read_f16(sh_ctx *ctx, const sh_paged_kv8 *kv, uint16_t *k, uint16_t *v, int tokens) {
  return read8<PagedF16>(ctx, kv, k, v, tokens);
}

SH_API int sh_paged8_read_bf16(sh_ctx *ctx, const sh_paged_kv8 *kv, uint16_t *k, uint16_t *v, int tokens) {
  return read8<PagedBf16>(ctx, kv, k, v, tokens);
}

}  // extern "C"
