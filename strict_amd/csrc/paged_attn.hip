// Attention of new tokens over a KV cache in pages (sh_attn_paged_*).
//
// A call is divided into equal pieces of work (paged.h): workgroup w takes the
// tiles of its piece, a tile being some tokens of one sequence with the query
// heads of one KV head, its rows (token, head) numbered token * G + head. A tile
// that lies in one piece is written to the output; one cut between pieces leaves
// a part in each of its workgroups' slots (V sums, maximum and sum of weights
// per row), and a second kernel merges the parts.
//
// Softmax runs over the positions in order with a running maximum, in base 2:
// s = q.k scale log2(e), weights 2^(s - max) (times 2^14 in fp16).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "llm_device.h"
#include "paged.h"
#include "paged_device.h"

namespace sh {
namespace {

constexpr int kT = 256;
constexpr int kWorkers = 512;

struct PagedAttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int *table;
  PagedPlan plan;
  MergeItem *items;  // [workers]
  float *slots;      // [2 workers][rows of a tile][d + 2]
  int heads, group, max_pages, num_pages, page_shift, tile_rows;
  float scale_log2;
};

// Row r of slot s: d V sums, then the row's maximum and sum of weights.
template <int kD>
__device__ __forceinline__ float *slot_row(const PagedAttnArgs &a, int slot, int r) {
  return a.slots + ((size_t)slot * a.tile_rows + r) * (kD + 2);
}

// Where the results of a tile's part go: the output (slot -1) or a slot.
template <class T, int kD>
__device__ __forceinline__ void store_value(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s,
                                            int slot, int r, int dim, float acc, float l) {
  if (slot < 0) {
    const size_t row = (size_t)(t.seq.row0 + s.first + r / a.group) * a.heads + t.kv_head * a.group + r % a.group;
    reinterpret_cast<typename T::Value *>(a.out)[row * kD + dim] = (typename T::Value)(l == 0.0f ? 0.0f : acc / l);
  } else {
    slot_row<kD>(a, slot, r)[dim] = acc;
  }
}

__device__ __forceinline__ float exp2_weight(float x) { return __builtin_amdgcn_exp2f(x); }

// Units [u0, u1) of a tile in fp32, a wave per row, a lane per position of 64:
// whatever the values are. A score of -infinity, and a weight that is 0 in fp32,
// adds nothing. Slow: for parts whose sums by MFMA are not finite.
template <class T, int kD>
__device__ void attn_exact(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s, int u0, int u1, int slot) {
  typedef typename T::Value Value;
  constexpr int kDims = kD / 64;
  const int lane = threadIdx.x & 63, rows = s.count * a.group;
  const Value *kp = reinterpret_cast<const Value *>(a.k), *vp = reinterpret_cast<const Value *>(a.v);
  for (int r = threadIdx.x >> 6; r < rows; r += kT / 64) {
    const int pos = s.pos0 + r / a.group;
    const Value *q = reinterpret_cast<const Value *>(a.q) +
                     ((size_t)(t.seq.row0 + s.first + r / a.group) * a.heads + t.kv_head * a.group + r % a.group) * kD;
    float m = -INFINITY, l = 0.0f, acc[kDims];
#pragma unroll
    for (int j = 0; j < kDims; j++) acc[j] = 0.0f;
    for (int u = u0; u < u1; u++) {
      const int p0 = span_position(s, a.plan.unit, u), end = min(p0 + a.plan.unit, s.hi);
      for (int pt = p0; pt < end; pt += 64) {
        const int p = pt + lane;
        bool seen = p < end && p <= pos && (a.plan.window == 0 || p > pos - a.plan.window || p < s.sinks);
        long long at = 0;  // of the position's k and v
        if (seen) {
          const int page = paged_page(a.table[(size_t)t.b * a.max_pages + (p >> a.page_shift)], a.num_pages);
          seen = page >= 0;
          at = (((((long long)max(page, 0) * a.plan.kv_heads + t.kv_head) << a.page_shift) +
                 (p & ((1 << a.page_shift) - 1))) * kD);
        }
        float sc = -INFINITY;
        if (seen) {
          float dot = 0.0f;
          for (int c = 0; c < kD; c++) dot = fmaf((float)q[c], (float)kp[at + c], dot);
          sc = dot * a.scale_log2;
        }
        const float top = fmaxf(m, wave_max(sc));
        const float w = sc == -INFINITY ? 0.0f : exp2_weight(sc - top + T::kWeightLog2);
        const float c = top == m ? 1.0f : exp2_weight(m - top);
        l = l * c + wave_sum(w);
        m = top;
#pragma unroll
        for (int j = 0; j < kDims; j++) acc[j] *= c;
        for (int i = 0; i < 64; i++) {
          const float wi = __shfl(w, i, 64);
          const long long ai = __shfl(at, i, 64);
          if (wi == 0.0f) continue;
#pragma unroll
          for (int j = 0; j < kDims; j++) acc[j] = fmaf(wi, (float)vp[ai + lane + 64 * j], acc[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kDims; j++) store_value<T, kD>(a, t, s, slot, r, lane + 64 * j, acc[j], l);
    if (slot >= 0 && lane == 0) {
      slot_row<kD>(a, slot, r)[kD] = m;
      slot_row<kD>(a, slot, r)[kD + 1] = l;
    }
  }
}

// Prefix sums of the sequences' costs, by threads of `per` sequences each.
__device__ __forceinline__ void scan_costs(const PagedPlan &p, int per, long long *prefix, long long *waves) {
  const int t = threadIdx.x, lane = t & 63;
  long long sum = 0;
  for (int b = t * per; b < min((t + 1) * per, p.batch); b++) sum = plan_add(sum, plan_cost(p, plan_seq(p, b)));
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const long long o = __shfl_up(sum, off, 64);
    if (lane >= off) sum = plan_add(sum, o);
  }
  if (lane == 63) waves[t >> 6] = sum;
  __syncthreads();
  for (int w = 0; w < (t >> 6); w++) sum = plan_add(sum, waves[w]);
  prefix[t + 1] = sum;
  if (t == 0) prefix[0] = 0;
  __syncthreads();
}

// A worker's piece, tile by tile: part(tile, span, u0, u1, slot).
template <class Part>
__device__ __forceinline__ void walk_piece(const PagedAttnArgs &a, int worker, Part part) {
  __shared__ long long prefix[kT + 1], waves[kT / 64];
  const PagedPlan &p = a.plan;
  const int per = (p.batch + kT - 1) / kT;
  scan_costs(p, per, prefix, waves);
  const long long total = prefix[kT], piece = plan_piece(p, total);
  const long long x0 = worker * piece, x1 = min(x0 + piece, total);
  MergeItem item = {0, 0, 0, 0, 0, 0};
  for (long long x = x0; x < x1;) {
    const PieceStep st = plan_step(p, prefix, kT, per, piece, worker, x0, x1, x, &item);
    if (!st.more) break;
    if (st.run) part(st.tile, st.span, st.u0, st.u1, st.slot);
    x = st.tile.begin + st.tile.cost;
  }
  if (threadIdx.x == 0) a.items[worker] = item;
}

template <class T, int kD>
__global__ __launch_bounds__(kT) void paged_attn_kernel(const PagedAttnArgs a) {
  const int worker = blockIdx.x;
  walk_piece(a, worker, [&](const PagedTile &t, const TileSpan &s, int u0, int u1, int slot) {
    attn_exact<T, kD>(a, t, s, u0, u1, slot);
  });
}

// grid (workers): the parts of the tile whose first inner cut is at this
// worker's start, against their common maximum. (A part that saw nothing, of
// maximum -infinity, has no weight.)
template <class T, int kD>
__global__ __launch_bounds__(kT) void paged_merge_kernel(const PagedAttnArgs a) {
  const MergeItem it = a.items[blockIdx.x];
  const int dim = threadIdx.x % kD;
  for (int r = threadIdx.x / kD; it.parts > 0 && r < it.tokens * a.group; r += kT / kD) {
    float top = -INFINITY, num = 0.0f, den = 0.0f;
    for (int j = 0; j < it.parts; j++) {
      const float *p = slot_row<kD>(a, j == 0 ? it.first_slot : 2 * (it.first_worker + j), r);
      const float m = p[kD], old = top;
      if (m == -INFINITY && p[kD + 1] == 0.0f) continue;
      top = fmaxf(top, m);
      const float c = old == top ? 1.0f : exp2_weight(old - top), w = m == top ? 1.0f : exp2_weight(m - top);
      num = num * c;
      den = den * c;
      if (w != 0.0f || p[kD + 1] != p[kD + 1]) {  // (a part of NaN scores stays NaN)
        num = fmaf(w, p[dim], num);
        den = fmaf(w, p[kD + 1], den);
      }
    }
    const size_t row = (size_t)(it.row0 + r / a.group) * a.heads + it.kv_head * a.group + r % a.group;
    reinterpret_cast<typename T::Value *>(a.out)[row * kD + dim] = (typename T::Value)(den == 0.0f ? 0.0f : num / den);
  }
}

// ---- the entry points ---------------------------------------------------------------

int tile_rows_of(int group) { return group <= 16 ? 16 : 128; }

size_t workspace_of(const sh_paged_kv *kv, int heads) {
  return (size_t)kWorkers * sizeof(MergeItem) +
         (size_t)2 * kWorkers * tile_rows_of(heads / kv->kv_heads) * (kv->head_dim + 2) * 4;
}

int check_attn_sizes(const sh_paged_kv *kv, int tokens, int heads, int max_new) {
  if (const char *wrong = check_paged_sizes(kv, tokens, heads)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (!paged_dim_built(kv->head_dim))
    return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", kv->head_dim);
  if (max_new < 0) return fail(SH_ERR_INVALID_ARGUMENT, "max_new must not be negative");
  return SH_OK;
}

template <class T>
int attn_paged(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *q, uint16_t *out, int tokens, int heads,
               int max_new, int window, int sinks, float scale, void *workspace, size_t workspace_bytes) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if ((rc = check_attn_sizes(kv, tokens, heads, max_new))) return rc;
  if (window < 0 || sinks < 0) return fail(SH_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return fail(SH_ERR_INVALID_ARGUMENT, "scale must be positive and finite");
  if (tokens == 0 || kv->batch == 0) return SH_OK;
  const size_t bytes = (size_t)tokens * heads * kv->head_dim * 2, need = workspace_of(kv, heads);
  if ((rc = check_paged_pointers(ctx, kv)) || (rc = check_range(ctx, q, bytes, "q")) ||
      (rc = check_range(ctx, out, bytes, "out")))
    return rc;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
  if (ranges_overlap(q, bytes, out, bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "out overlaps q");
  if (workspace_bytes < need)
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer has %zu bytes, %zu are needed", workspace_bytes, need);
  if ((rc = check_range(ctx, workspace, need, "workspace"))) return rc;
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer must be 16-byte aligned");
  PagedAttnArgs a;
  a.q = q;
  a.k = kv->k;
  a.v = kv->v;
  a.out = out;
  a.table = kv->page_table;
  a.heads = heads;
  a.group = heads / kv->kv_heads;
  a.max_pages = kv->max_pages;
  a.num_pages = kv->num_pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  a.tile_rows = tile_rows_of(a.group);
  a.scale_log2 = scale * 1.44269504f;
  a.items = static_cast<MergeItem *>(workspace);
  a.slots = reinterpret_cast<float *>(a.items + kWorkers);
  PagedPlan &p = a.plan;
  p.starts = kv->starts;
  p.lengths = kv->lengths;
  p.batch = kv->batch;
  p.tokens = tokens;
  p.kv_heads = kv->kv_heads;
  p.capacity = kv->max_pages * kv->page_size;
  p.per_tile = a.tile_rows / a.group;
  p.unit = 64;
  p.window = window;
  p.sinks = sinks;
  p.workers = kWorkers;
  p.min_piece = 256;
  p.whole_below = 0;
  const hipStream_t st = stream_of(ctx);
  if (kv->head_dim == 64) {
    paged_attn_kernel<T, 64><<<kWorkers, kT, 0, st>>>(a);
    paged_merge_kernel<T, 64><<<kWorkers, kT, 0, st>>>(a);
  } else {
    paged_attn_kernel<T, 128><<<kWorkers, kT, 0, st>>>(a);
    paged_merge_kernel<T, 128><<<kWorkers, kT, 0, st>>>(a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "attn_paged");
}

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_attn_paged_workspace(const sh_paged_kv *kv, int tokens, int heads, int max_new, size_t *bytes) {
  if (!bytes) return fail(SH_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const int rc = check_attn_sizes(kv, tokens, heads, max_new);
  if (rc != SH_OK) return rc;
  *bytes = workspace_of(kv, heads);
  return SH_OK;
}

SH_API int sh_attn_paged_f16(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *q, uint16_t *out, int tokens,
                             int heads, int max_new, int window, int sinks, float scale, void *workspace,
                             size_t workspace_bytes) {
  return attn_paged<PagedF16>(ctx, kv, q, out, tokens, heads, max_new, window, sinks, scale, workspace,
                              workspace_bytes);
}

SH_API int sh_attn_paged_bf16(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *q, uint16_t *out, int tokens,
                              int heads, int max_new, int window, int sinks, float scale, void *workspace,
                              size_t workspace_bytes) {
  return attn_paged<PagedBf16>(ctx, kv, q, out, tokens, heads, max_new, window, sinks, scale, workspace,
                               workspace_bytes);
}

}  // extern "C"
