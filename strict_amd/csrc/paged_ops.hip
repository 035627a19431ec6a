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

// cos and sin of an fp64 angle below 2^29 (check_rope_theta) to fp32: reduction by pi / 2 in two
// parts (Cody and Waite) and Taylor polynomials on [-pi / 4, pi / 4], in fp64.
__device__ __forceinline__ void cos_sin64(double a, float *c, float *s) {
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
  *s = (float)((k & 2) ? -sd : sd);
  *c = (float)((k == 1 || k == 2) ? -cd : cd);
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
    float x1[8], x2[8], ss = 0.0f;
    unpack8<T>(lo[u], x1);
    unpack8<T>(hi[u], x2);
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
#pragma unroll
    for (int off = 1; off < kLanes; off *= 2) ss += __shfl_xor(ss, off, 64);
    const float inv = 1.0f / sqrtf(ss * (1.0f / kD) + a.eps);
    const float *gain = (is_q ? a.q_gain : a.k_gain) + part * 8;
    u32x4 o1 = lo[u], o2 = hi[u];
    if (is_q || is_k) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float y1 = x1[e] * inv * gain[e], y2 = x2[e] * inv * gain[e + kHalf];
        x1[e] = y1 * f[e].x - y2 * f[e].y;
        x2[e] = y2 * f[e].x + y1 * f[e].y;
      }
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
  for (int i = 0; i < d / 2; i++) a.freq[i] = std::pow((double)theta, -2.0 * i / d);
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
