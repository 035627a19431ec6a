// What goes into a KV cache in pages: the head norms and RoPE of new tokens with
// their k and v stored in pages, and copies of pages (the cache's layout: paged.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "paged.h"
#include "paged_device.h"

namespace sh {
namespace {

constexpr int kT = 256;

// ---- head norms, RoPE and the pages ------------------------------------------------

struct NormRopeArgs {
  const uint16_t *qkv;
  const float *q_gain, *k_gain;
  uint16_t *q, *k, *v;
  const int *table, *lengths, *starts;
  int tokens, batch, max_pages, num_pages, page_shift, heads, kv_heads, ld, chunks;
  float eps;
  double freq[64];  // theta^(-2i / d)
};

// A wave takes 4 * kHeadsAt heads of one token: q heads, then k, then v. A head is
// d / 16 lanes wide, 8 values of its first half and the 8 that rotate with them in
// each lane, all loads requested at once. The factors, one pair of them per lane,
// are worked out meanwhile and go round through LDS. Bound by the rows' bytes: 152 MB
// of bf16 rows of 32 heads of 128 in and out in 25 us, 6.0 TB/s. (Stores that the
// caches need not keep: 36 us with ordinary ones. Loads of that kind as well: 28.)
template <class T, int kD>
__global__ __launch_bounds__(kT) void norm_rope_kernel(const NormRopeArgs a) {
  constexpr int kLanes = kD / 16, kHeadsAt = 64 / kLanes, kSteps = 4, kHalf = kD / 2;
  __shared__ float2 factors[kT / 64][kHalf];
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
  const int b = find_seq(a.starts, a.batch, row);
  if (b < 0 || b >= a.batch) return;  // a row of no sequence
  const PagedSeq s = paged_seq(a.starts[b], a.starts[b + 1], a.lengths[b], a.tokens, a.max_pages << a.page_shift);
  const int pos = s.len - s.n + (row - s.row0);
  if (lane < kHalf) {
    float c, sn;
    cos_sin64((double)pos * a.freq[lane], &c, &sn);
    factors[wave][lane] = make_float2(c, sn);
  }
  __builtin_amdgcn_wave_barrier();
  float2 f[8];
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = factors[wave][part * 8 + e];
  int page = -1;
  if (pos >= 0 && pos < s.len) page = paged_page(a.table[(size_t)b * a.max_pages + (pos >> a.page_shift)], a.num_pages);
  const int in_page = pos & ((1 << a.page_shift) - 1);
#pragma unroll
  for (int u = 0; u < kSteps; u++) {
    const int h = h0 + u * kHeadsAt + sub;
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    u32x4 o1 = lo[u], o2 = hi[u];
    if (is_q || is_k) {
      float x1[8], x2[8];
      unpack8<T>(lo[u], x1);
      unpack8<T>(hi[u], x2);
      head_norm_rope<kD>(x1, x2, (is_q ? a.q_gain : a.k_gain) + part * 8, a.eps, [&](int e) { return f[e]; });
      o1 = pack8<T>(x1);
      o2 = pack8<T>(x2);
    }
    if (h >= all || (!is_q && page < 0)) continue;
    uint16_t *to;
    if (is_q)
      to = a.q + ((size_t)row * a.heads + h) * kD;
    else
      to = (is_k ? a.k : a.v) +
           ((((size_t)page * a.kv_heads + (h - a.heads - (is_k ? 0 : a.kv_heads))) << a.page_shift) + in_page) * kD;
    __builtin_nontemporal_store(o1, reinterpret_cast<u32x4 *>(to + part * 8));
    __builtin_nontemporal_store(o2, reinterpret_cast<u32x4 *>(to + part * 8 + kHalf));
  }
}

template <class T>
int norm_rope(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *qkv, const float *q_gain,
              const float *k_gain, uint16_t *q, int tokens, int heads, int ld, float eps, float theta) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (const char *wrong = check_paged_sizes(kv, tokens, heads)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  const int d = kv->head_dim;
  if (!paged_dim_built(d)) return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", d);
  if (!(eps >= 0.0f)) return fail(SH_ERR_INVALID_ARGUMENT, "eps must be >= 0");
  if (const char *wrong = check_rope_theta(kv, tokens, theta)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  const long long width = ((long long)heads + 2LL * kv->kv_heads) * d;
  if (ld < width || ld % 8 != 0)
    return fail(SH_ERR_INVALID_ARGUMENT, "ld %d must be a multiple of 8 and at least %lld", ld, width);
  if (tokens == 0 || kv->batch == 0) return SH_OK;
  const size_t in_bytes = ((size_t)(tokens - 1) * ld + (size_t)width) * 2, q_bytes = (size_t)tokens * heads * d * 2;
  if ((rc = check_paged_pointers(ctx, kv)) || (rc = check_range(ctx, qkv, in_bytes, "qkv")) ||
      (rc = check_range(ctx, q_gain, (size_t)d * 4, "q_gain")) ||
      (rc = check_range(ctx, k_gain, (size_t)d * 4, "k_gain")) || (rc = check_range(ctx, q, q_bytes, "q")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "qkv and q must be 16-byte aligned");
  if (ranges_overlap(qkv, in_bytes, q, q_bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "q overlaps qkv");
  const size_t pool = paged_pool_bytes(kv);
  if (ranges_overlap(kv->k, pool, kv->v, pool)) return fail(SH_ERR_INVALID_ARGUMENT, "the k and v pages overlap");
  if (ranges_overlap(kv->k, pool, q, q_bytes) || ranges_overlap(kv->v, pool, q, q_bytes) ||
      ranges_overlap(kv->k, pool, qkv, in_bytes) || ranges_overlap(kv->v, pool, qkv, in_bytes))
    return fail(SH_ERR_INVALID_ARGUMENT, "the cache overlaps q or qkv");
  const size_t gain_bytes = (size_t)d * 4;
  const auto over_inputs = [&](const void *p, size_t bytes) {
    return overlaps_index(kv, p, bytes) || ranges_overlap(p, bytes, q_gain, gain_bytes) ||
           ranges_overlap(p, bytes, k_gain, gain_bytes);
  };
  if (over_inputs(q, q_bytes) || over_inputs(kv->k, pool) || over_inputs(kv->v, pool))
    return fail(SH_ERR_INVALID_ARGUMENT, "q or the cache overlaps the page table, lengths, starts or gains");
  NormRopeArgs a;
  a.qkv = qkv;
  a.q_gain = q_gain;
  a.k_gain = k_gain;
  a.q = q;
  a.k = kv->k;
  a.v = kv->v;
  a.table = kv->page_table;
  a.lengths = kv->lengths;
  a.starts = kv->starts;
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
  const int per_unit = 4 * (64 / (d / 16));
  a.chunks = (heads + 2 * kv->kv_heads + per_unit - 1) / per_unit;
  const long long units = (long long)tokens * a.chunks;
  const unsigned grid = (unsigned)((units + kT / 64 - 1) / (kT / 64));
  if (d == 64)
    norm_rope_kernel<T, 64><<<grid, kT, 0, stream_of(ctx)>>>(a);
  else
    norm_rope_kernel<T, 128><<<grid, kT, 0, stream_of(ctx)>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "qk_norm_rope_paged");
}

// ---- page copies ----------------------------------------------------------------------

constexpr int kCopyVectors = 4;  // of 16 bytes per thread

// grid (chunks of a page, pages, planes): 16 KiB of one page, all of a thread's
// loads requested before its first store. Bound by the bytes: 257 MB both ways in 45 us,
// 5.7 TB/s (as accesses that the caches keep: 51).
__global__ __launch_bounds__(kT) void pages_copy_kernel(uint8_t *pool, size_t plane_stride, int num_pages,
                                                        uint32_t page_vectors, int chunks,
                                                        const int *__restrict__ src,
                                                        const int *__restrict__ dst) {
  const int i = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int from = paged_page(src[i], num_pages), to = paged_page(dst[i], num_pages);
  if (from < 0 || to < 0 || from == to) return;
  u32x4 *plane = reinterpret_cast<u32x4 *>(pool + blockIdx.y * plane_stride);
  const u32x4 *s = plane + (size_t)from * page_vectors;
  u32x4 *d = plane + (size_t)to * page_vectors;
  const uint32_t at = (uint32_t)chunk * (kT * kCopyVectors) + threadIdx.x;
  u32x4 v[kCopyVectors];
#pragma unroll
  for (int u = 0; u < kCopyVectors; u++) v[u] = __builtin_nontemporal_load(s + min(at + u * kT, page_vectors - 1));
#pragma unroll
  for (int u = 0; u < kCopyVectors; u++)
    if (at + u * kT < page_vectors) __builtin_nontemporal_store(v[u], d + at + u * kT);
}

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_qk_norm_rope_paged_f16(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *qkv,
                                     const float *q_gain, const float *k_gain, uint16_t *q, int tokens,
                                     int heads, int ld, float eps, float theta) {
  return norm_rope<PagedF16>(ctx, kv, qkv, q_gain, k_gain, q, tokens, heads, ld, eps, theta);
}

SH_API int sh_qk_norm_rope_paged_bf16(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *qkv,
                                      const float *q_gain, const float *k_gain, uint16_t *q, int tokens,
                                      int heads, int ld, float eps, float theta) {
  return norm_rope<PagedBf16>(ctx, kv, qkv, q_gain, k_gain, q, tokens, heads, ld, eps, theta);
}

SH_API int sh_pages_copy(sh_ctx *ctx, void *pool, int planes, size_t plane_stride, int num_pages,
                         size_t page_bytes, const int32_t *src, const int32_t *dst, int count) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if (const char *wrong = check_pages_copy(planes, plane_stride, num_pages, page_bytes, count))
    return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (planes == 0 || count == 0) return SH_OK;
  const size_t extent = (planes - 1) * plane_stride + (size_t)num_pages * page_bytes;
  if ((rc = check_range(ctx, pool, extent, "pool")) || (rc = check_range(ctx, src, (size_t)count * 4, "src")) ||
      (rc = check_range(ctx, dst, (size_t)count * 4, "dst")))
    return rc;
  if (reinterpret_cast<uintptr_t>(pool) & 15) return fail(SH_ERR_INVALID_ARGUMENT, "pool must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 3)  // (scalar loads)
    return fail(SH_ERR_INVALID_ARGUMENT, "src and dst must be 4-byte aligned");
  if (ranges_overlap(pool, extent, src, (size_t)count * 4) || ranges_overlap(pool, extent, dst, (size_t)count * 4))
    return fail(SH_ERR_INVALID_ARGUMENT, "src or dst lies in the pools");
  const uint32_t vectors = (uint32_t)(page_bytes / 16);
  const int chunks = (int)((vectors + kT * kCopyVectors - 1) / (kT * kCopyVectors));
  // (a launch takes fewer than 2^32 threads: 2^24 workgroups; a page is 2^17 of them at most)
  const int most = (1 << 24) - 1;
  for (int i0 = 0; i0 < count;) {
    const int pages = std::min(count - i0, most / chunks), blocks = pages * chunks;
    for (int p0 = 0; p0 < planes;) {
      const int n = std::min(planes - p0, most / blocks);
      pages_copy_kernel<<<dim3((unsigned)blocks, (unsigned)n), kT, 0, stream_of(ctx)>>>(
          static_cast<uint8_t *>(pool) + p0 * plane_stride, plane_stride, num_pages, vectors, chunks, src + i0, dst + i0);
      p0 += n;
    }
    i0 += pages;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "pages_copy");
}

}  // extern "C"
