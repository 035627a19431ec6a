// Attention of new tokens over a KV cache in pages (sh_attn_paged_*).
//
// A call is divided into equal pieces of work (paged.h): workgroup w takes the
// tiles of its piece, a tile being some tokens of one sequence with the query
// heads of one KV head, its rows (token, head) numbered token * G + head. A tile
// that lies in one piece is written to the output; one cut between pieces leaves
// a part in each of its workgroups' slots (V sums, maximum and sum of weights
// per row), and a second kernel merges the parts. That kernel also works out again,
// in fp32 without matrix products, what came out not finite: infinities and NaN in
// q, K or V, or in places of V that only some of a tile's rows see.
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

constexpr int kT = 256, kMaxT = 512;
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define SH_PAGED_LDS __attribute__((address_space(3)))

// Pieces of a call, and the shortest, in positions: three workgroups per CU are
// resident with the small tiles, two with the large ones.
constexpr int kSmallRows = 16, kSmallWorkers = 512, kSmallPiece = 128, kSmallWhole = 192, kSmallMergeRows = 1;
constexpr int kLargeRows = 128, kLargeWorkers = 512, kLargePiece = 256, kLargeWhole = 1400, kLargeMergeRows = 8;

struct PagedAttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int *table;
  PagedPlan plan;
  MergeItem *items;  // [workers]
  int *groups;       // [workers]: rows to merge of the worker's item, in groups
  int *redo;         // [workers]: 1: some of the worker's results are not finite
  float *slots;      // [2 workers][rows of a tile][d + 4]
  int heads, group, group_inv, max_pages, num_pages, page_shift, tile_rows;
  float scale_log2;
};

// Token of a tile's row (r <= 255, group <= 128: exact), and its row of heads in q
// and out.
__device__ __forceinline__ int token_of(const PagedAttnArgs &a, int r) { return (r * a.group_inv) >> 16; }
__device__ __forceinline__ size_t head_row(const PagedAttnArgs &a, int row0, int kv_head, int r) {
  const int token = token_of(a, r);
  return (size_t)(row0 + token) * a.heads + kv_head * a.group + (r - token * a.group);
}

// Row r of slot s: d V sums, then the row's maximum and sum of weights (and 8
// bytes that align the next).
template <int kD>
__device__ __forceinline__ float *slot_row(const PagedAttnArgs &a, int slot, int r) {
  return a.slots + ((size_t)slot * a.tile_rows + r) * (kD + 4);
}

// Where the results of a tile's part go: the output (slot -1) or a slot.
template <class T, int kD>
__device__ __forceinline__ void store_value(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s,
                                            int slot, int r, int dim, float acc, float l) {
  if (slot < 0) {
    const size_t row = head_row(a, t.seq.row0 + s.first, t.kv_head, r);
    reinterpret_cast<typename T::Value *>(a.out)[row * kD + dim] = (typename T::Value)(l == 0.0f ? 0.0f : acc / l);
  } else {
    slot_row<kD>(a, slot, r)[dim] = acc;
  }
}

__device__ __forceinline__ float exp2_weight(float x) { return __builtin_amdgcn_exp2f(x); }

// A tile in fp32, a wave per row, a lane per position of 64:
// whatever the values are. A score of -infinity, and a weight that is 0 in fp32,
// adds nothing. Slow: for tiles whose sums by MFMA are not finite.
template <class T, int kD>
__device__ void attn_exact(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s) {
  typedef typename T::Value Value;
  constexpr int kDims = kD / 64;
  const int lane = threadIdx.x & 63, rows = s.count * a.group;
  const Value *kp = reinterpret_cast<const Value *>(a.k), *vp = reinterpret_cast<const Value *>(a.v);
  for (int r = threadIdx.x >> 6; r < rows; r += blockDim.x >> 6) {
    const int pos = s.pos0 + token_of(a, r);
    const Value *q = reinterpret_cast<const Value *>(a.q) + head_row(a, t.seq.row0 + s.first, t.kv_head, r) * kD;
    float m = -INFINITY, l = 0.0f, acc[kDims];
#pragma unroll
    for (int j = 0; j < kDims; j++) acc[j] = 0.0f;
    for (int u = 0; u < s.units; u++) {
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
    for (int j = 0; j < kDims; j++) store_value<T, kD>(a, t, s, -1, r, lane + 64 * j, acc[j], l);
  }
}

// The line's division among the workers, in LDS.
struct PlanLds {
  long long prefix[kT + 1], waves[kMaxT / 64];
  PlanSeq seqs[kT];  // where a thread has one sequence
};

// Prefix sums of the sequences' costs, by kT threads (of kT or more) of `per`
// sequences each.
__device__ __forceinline__ void scan_costs(const PagedPlan &p, int per, PlanLds &lds) {
  const int t = threadIdx.x, lane = t & 63;
  long long sum = 0;
  for (int b = t * per; b < min((t + 1) * per, p.batch); b++) {
    const PlanSeq s = plan_sequence(p, b);
    if (per == 1) lds.seqs[t] = s;
    sum = plan_add(sum, s.one * p.kv_heads);
  }
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const long long o = __shfl_up(sum, off, 64);
    if (lane >= off) sum = plan_add(sum, o);
  }
  if (lane == 63) lds.waves[t >> 6] = sum;
  __syncthreads();
  for (int w = 0; w < (t >> 6); w++) sum = plan_add(sum, lds.waves[w]);
  if (t < kT) lds.prefix[t + 1] = sum;
  if (t == 0) lds.prefix[0] = 0;
  __syncthreads();
}

// The last i < kT with prefix[i] <= x: how many of the values from prefix[1] on are
// (a wave looks at all 256 at once).
__device__ __forceinline__ int find_part(const PlanLds &lds, long long x) {
  const int lane = threadIdx.x & 63;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; i++) n += __popcll(__ballot(lds.prefix[1 + i * 64 + lane] <= x));
  return min(n, kT - 1);
}

// A worker's piece, step by step: part(step), which says whether its results are
// finite. Returns whether all are.
template <class Part>
__device__ __forceinline__ bool walk_piece(const PagedPlan &p, int worker, PlanLds &lds, MergeItem *item,
                                           long long *piece_out, Part part) {
  const int per = (p.batch + kT - 1) / kT;
  scan_costs(p, per, lds);
  const long long total = lds.prefix[kT], piece = plan_piece(p, total);
  const long long x0 = worker * piece, x1 = min(x0 + piece, total);
  *piece_out = piece;
  bool finite = true;
  for (long long x = x0; x < x1;) {
    const int i = find_part(lds, x);
    const PagedTile t = plan_locate(p, lds.seqs, i, per, lds.prefix[i], x);
    const PieceStep st = plan_step(p, t, piece, worker, x0, x, item);
    if (!st.more) break;
    if (st.run && !part(st)) finite = false;
    x = t.begin + t.cost;
  }
  return finite;
}

// A worker of the main kernels.
template <int kMergeRows, class Part>
__device__ __forceinline__ void work_piece(const PagedAttnArgs &a, int worker, PlanLds &lds, Part part) {
  MergeItem item = {0, 0, 0, 0, 0, 0};
  long long piece;
  const bool finite = walk_piece(a.plan, worker, lds, &item, &piece, part);
  if (threadIdx.x == 0) {
    a.items[worker] = item;
    a.groups[worker] = item.parts > 0 ? (item.tokens * a.group + kMergeRows - 1) / kMergeRows : 0;
    a.redo[worker] = finite ? 0 : 1;
  }
}

__device__ __forceinline__ void wait_lds() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): loads from memory stay in flight
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
__device__ __forceinline__ void lds_barrier() {
  wait_lds();
  __builtin_amdgcn_s_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// Whether token position `pos` sees position p of the tile's span.
__device__ __forceinline__ bool sees(const PagedAttnArgs &a, const TileSpan &s, int pos, int p) {
  return p <= pos && (a.plan.window == 0 || p > pos - a.plan.window || p < s.sinks);
}
// Whether any token of the tile does.
__device__ __forceinline__ bool tile_sees(const PagedAttnArgs &a, const TileSpan &s, int p) {
  return p < s.hi && (a.plan.window == 0 || p >= s.lo || p < s.sinks);
}

// The larger of a lane's value and lane ^ 32's. (Asm: of the builtin's two results
// the compiler keeps one, taking them for equal. The operands need to have been
// written two states before.)
__device__ __forceinline__ float half_max(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}

// ---- tiles of up to 16 rows ------------------------------------------------------------
//
// One token of a sequence (or a few) with the G query heads of a KV head: bound by
// the K and V bytes. Each wave takes units of 32 positions (64 at head_dim 64) by
// itself, all of a unit's loads requested before any is used and the next unit's as
// soon as registers are free, and keeps a running softmax of its own; the four are
// combined at the end. Rows in the columns of the matrix products:
//  - scores as K x q: K fragments straight from memory (a lane: 8 dims of position
//    lane % 16); a lane then holds 4 consecutive positions of each 16 for its row;
//  - V sums as V^T x P, the k slots numbered as P has them (slot (g, e): position
//    4 g + e of the first 16 for e < 4, of the second for e >= 4); V goes through
//    LDS rows as it is and comes back by transposing reads.
// A unit's 16-position blocks lie in one page each (pages of 16 and more).
template <int kD>
constexpr int kSmallUnit = 32 * 128 / kD;

template <class T, int kD>
struct SmallLds {
  union {
    uint8_t v[4][kSmallUnit<kD> * kD * 2];
    float acc[4][kSmallRows][kD];
  };
  float stat[4][kSmallRows][2];
};

template <class T, int kD>
__device__ __forceinline__ bool attn_small(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s, int u0,
                                           int u1, int slot, SmallLds<T, kD> &lds) {
  typedef typename T::Vec Vec;
  typedef typename T::Value Value;
  constexpr int kUnit = kSmallUnit<kD>, kBlocks = kUnit / 16, kKK = kD / 32, kDT = kD / 16;
  constexpr int kRow = kD * 2, kChunks = kD / 8, kVLoads = kUnit * kChunks / 64, kVRows = 64 / kChunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, grp = lane >> 4, rows = s.count * a.group;
  const int row = min(r16, rows - 1), my_pos = s.pos0 + token_of(a, row);
  const uint16_t *qp = a.q + head_row(a, t.seq.row0 + s.first, t.kv_head, row) * kD + grp * 8;
  const int *table = a.table + (size_t)t.b * a.max_pages;
  const int last_pos = s.pos0 + s.count - 1, page_mask = (1 << a.page_shift) - 1;
  Vec q[kKK];
#pragma unroll
  for (int kk = 0; kk < kKK; kk++) q[kk] = *reinterpret_cast<const Vec *>(qp + 32 * kk);

  // the table entry of block lane % kBlocks of unit j
  auto entry = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kUnit, min(j, u1 - 1)) + 16 * (lane % kBlocks);
    return table[min(p >> a.page_shift, a.max_pages - 1)];
  };
  Vec kf[kBlocks][kKK];
  u32x4 vr[kVLoads];
  size_t base[kBlocks];  // of the blocks' first rows, in values; bad: no page
  auto place = [&](int j, int entries, unsigned *bad) __attribute__((always_inline)) {
    const int p = span_position(s, kUnit, j);
    *bad = 0;
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++) {
      const int page = paged_page(__builtin_amdgcn_readlane(entries, tt), a.num_pages);
      if (page < 0) *bad |= 1u << tt;
      base[tt] = ((((size_t)max(page, 0) * a.plan.kv_heads + t.kv_head) << a.page_shift) + ((p + 16 * tt) & page_mask)) * kD;
    }
  };
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
      for (int kk = 0; kk < kKK; kk++)
        kf[tt][kk] = *reinterpret_cast<const Vec *>(a.k + base[tt] + (r16 * kD + grp * 8 + 32 * kk));
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kVLoads; u++)
      vr[u] = *reinterpret_cast<const u32x4 *>(
          a.v + base[u * kVRows / 16] + ((u * kVRows % 16 + lane / kChunks) * kD + (lane % kChunks) * 8));
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x4 acc[kDT];
#pragma unroll
  for (int dt = 0; dt < kDT; dt++) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint8_t *vl = lds.v[wave];
  // chunk c of row r lies at c ^ f(r): a transposing read's 32 lanes (8 rows, 2
  // chunks each) then hit 64 banks
  auto swz = [](int r) { return kD == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); };
  const int ti = (lane >> 2) & 3, tq = lane & 3;
  int v_to[2], v_at[kDT];  // (f repeats every 8 rows)
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int r = u * kVRows + lane / kChunks;
    v_to[u] = r * kRow + (((lane % kChunks) ^ swz(r)) * 16);
  }
#pragma unroll
  for (int dt = 0; dt < kDT; dt++) {
    const int r = 4 * grp + ti;
    v_at[dt] = r * kRow + (((2 * dt + (tq >> 1)) ^ swz(r)) * 16) + (tq & 1) * 8;
  }
  auto unit = [&](int j, unsigned bad, unsigned *next_bad, int *entries) __attribute__((always_inline)) {
    const int p0 = span_position(s, kUnit, j), next = j + 4;
    f32x4 sc[kBlocks];
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++) sc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < kKK; kk++)
#pragma unroll
      for (int tt = 0; tt < kBlocks; tt++) sc[tt] = T::mfma16(kf[tt][kk], q[kk], sc[tt]);
    if (next < u1) {
      place(next, *entries, next_bad);
      __builtin_amdgcn_sched_barrier(0);
      load_k();
      __builtin_amdgcn_sched_barrier(0);
    }
    // every row sees every position
    const bool plain = bad == 0 && p0 + kUnit <= s.pos0 + 1 &&
                       (a.plan.window == 0 || p0 > last_pos - a.plan.window || p0 + kUnit <= s.sinks);
    // V to this wave's LDS rows (LDS works in order: after the last unit's reads);
    // what no row sees as zeros
    if (!plain) {
#pragma unroll
      for (int u = 0; u < kVLoads; u++)
        if (((bad >> (u * kVRows / 16)) & 1) || !tile_sees(a, s, p0 + u * kVRows + lane / kChunks))
          vr[u] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < kVLoads; u++) {
      *reinterpret_cast<u32x4 *>(vl + v_to[u & 1] + (u & ~1) * kVRows * kRow) = vr[u];
    }
    if (next < u1) {
      __builtin_amdgcn_sched_barrier(0);
      load_v();
      *entries = entry(next + 4);
      __builtin_amdgcn_sched_barrier(0);
    }
    float mx = -INFINITY;
    if (!plain) {
#pragma unroll
      for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (((bad >> tt) & 1) || !sees(a, s, my_pos, p0 + 16 * tt + 4 * grp + e)) sc[tt][e] = -INFINITY;
        }
    }
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
      for (int e = 0; e < 4; e++) mx = fmaxf(mx, sc[tt][e]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2;
    const float m = fmaxf(m_run, mx);
    const float corr = m_run == m ? 1.0f : exp2_weight(m_run - m);
    m_run = m;
    // (a row that has seen nothing yet: its weights are exp2(-infinity))
    const float off = (m == -INFINITY ? 0.0f : m) - T::kWeightLog2;
    float ls = 0.0f;
    Vec p[kBlocks / 2];
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float w = exp2_weight(fmaf(sc[tt][e], a.scale_log2, -off));
        p[tt / 2][(tt & 1) * 4 + e] = (Value)w;
        ls += w;
      }
    l_run = l_run * corr + ls;  // this lane's positions; the groups are summed at the end
#pragma unroll
    for (int dt = 0; dt < kDT; dt++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[dt][e] *= corr;
    wait_lds();  // this wave's V rows are in LDS
#pragma unroll
    for (int sl = 0; sl < kBlocks / 2; sl++)
#pragma unroll
      for (int dt = 0; dt < kDT; dt++) {
        s16x4 half[2];
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++)
          half[q2] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (SH_PAGED_LDS s16x4 *)((SH_PAGED_LDS uint8_t *)vl + v_at[dt] + (32 * sl + 16 * q2) * kRow));
        const Vec vf = __builtin_bit_cast(Vec, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[dt] = T::mfma16(vf, p[sl], acc[dt]);
      }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  if (u0 + wave < u1) {
    unsigned bad = 0, next_bad = 0;
    int entries = entry(u0 + wave);
    place(u0 + wave, entries, &bad);
    load_k();
    load_v();
    entries = entry(u0 + wave + 4);
    for (int j = u0 + wave; j < u1; j += 4) {
      unit(j, bad, &next_bad, &entries);
      bad = next_bad;
    }
  }
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (grp == 0) {
    lds.stat[wave][r16][0] = m_run;
    lds.stat[wave][r16][1] = l_run;
  }
  lds_barrier();  // every wave's V reads are done: lds.v becomes lds.acc
  if (r16 < rows) {
#pragma unroll
    for (int dt = 0; dt < kDT; dt++) *reinterpret_cast<f32x4 *>(&lds.acc[wave][r16][16 * dt + 4 * grp]) = acc[dt];
  }
  lds_barrier();
  bool finite = true;
  for (int i = tid; i < rows * kD; i += kT) {
    const int r = i / kD, dim = i % kD;
    float m = lds.stat[0][r][0];
#pragma unroll
    for (int w = 1; w < 4; w++) m = fmaxf(m, lds.stat[w][r][0]);
    float sum = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = lds.stat[w][r][0] == m ? 1.0f : exp2_weight(lds.stat[w][r][0] - m);
      sum = fmaf(f, lds.acc[w][r][dim], sum);
      l = fmaf(f, lds.stat[w][r][1], l);
    }
    finite = finite && __builtin_fabsf(sum) < INFINITY && l < INFINITY;
    store_value<T, kD>(a, t, s, slot, r, dim, sum, l);
    if (slot >= 0 && dim == 0) {
      slot_row<kD>(a, slot, r)[kD] = m;
      slot_row<kD>(a, slot, r)[kD + 1] = l;
    }
  }
  return !__syncthreads_or(finite ? 0 : 1);
}

template <class T, int kD>
__global__ __launch_bounds__(kT, kSmallWorkers / 256) void paged_small_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) SmallLds<T, kD> lds;
  __shared__ PlanLds plan;
  work_piece<kSmallMergeRows>(a, blockIdx.x, plan, [&](const PieceStep &st) { return attn_small<T, kD>(a, st.tile, st.span, st.u0, st.u1, st.slot, lds); });
}

// ---- tiles of up to 128 rows ------------------------------------------------------------
//
// Chunks of many tokens: bound by the matrix products and the softmax between them.
// Four waves of 32 rows share K and V units of 64 positions in LDS, double-buffered
// and loaded straight into it, a barrier per unit. Rows in the columns again, so that
// a row's scores lie in two lanes and its maximum, sum and rescaling stay there:
//  - scores as K x q, 32 x 32 positions and rows, K fragments from LDS;
//  - V sums as V^T x P with the k slots numbered as P has them (slot (h, e) of 16
//    positions: 4 h + e for e < 4, 8 + 4 h + e - 4 after that), V by transposing reads.
// A wave skips the units that none of its rows sees.
constexpr int kLargeUnit = 64;
constexpr float kSlack = 8.0f;

template <int kD>
struct LargeLds {
  uint8_t k[2][kLargeUnit * kD * 2], v[2][kLargeUnit * kD * 2];
  __attribute__((aligned(16))) unsigned bad[2][4];  // a 16-position block without a page
};

template <class T, int kD>
__device__ __forceinline__ bool attn_large(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s, int u0,
                                           int u1, int slot, LargeLds<kD> &lds) {
  typedef typename T::Vec Vec;
  typedef typename T::Value Value;
  typedef Value Quad __attribute__((ext_vector_type(4)));
  constexpr int kRow = kD * 2, kChunks = kD / 8, kKK = kD / 16, kDB = kD / 32;
  constexpr int kLoadRows = 64 / kChunks, kLoads = 16 / kLoadRows;  // of a wave's 16 positions
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5, rows = s.count * a.group;
  const bool active = 32 * wave < rows;  // (of the wave)
  const int row = min(32 * wave + n32, rows - 1), my_pos = s.pos0 + token_of(a, row);
  const int pos_lo = s.pos0 + token_of(a, min(32 * wave, rows - 1));
  const int pos_hi = s.pos0 + token_of(a, min(32 * wave + 31, rows - 1));
  const int *table = a.table + (size_t)t.b * a.max_pages;
  const int page_mask = (1 << a.page_shift) - 1;
  const uint16_t *qp = a.q + head_row(a, t.seq.row0 + s.first, t.kv_head, row) * kD + h * 8;
  Vec q[kKK];
#pragma unroll
  for (int kk = 0; kk < kKK; kk++) q[kk] = *reinterpret_cast<const Vec *>(qp + 16 * kk);

  // chunk c of row r lies at c ^ f(r): 16 lanes that read one chunk of 16 rows of K
  // hit all banks, and 32 lanes of a transposing read of V (4 rows, 4 chunks each)
  auto swz_k = [](int r) { return kD == 128 ? r & 15 : (r >> 1) & 7; };
  auto swz_v = [](int r) { return kD == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; u++) {
    const int r = u * kLoadRows + lane / kChunks, c = lane % kChunks;
    k_off[u] = r * kRow + ((c ^ swz_k(r)) * 16);
    v_off[u] = r * kRow + ((c ^ swz_v(r)) * 16);
  }
  const uint32_t k_lds = (uint32_t)(uintptr_t)(SH_PAGED_LDS uint8_t *)lds.k[0];
  const uint32_t v_lds = (uint32_t)(uintptr_t)(SH_PAGED_LDS uint8_t *)lds.v[0];
  constexpr uint32_t kBuffer = kLargeUnit * kD * 2, kWave = 16 * kRow;
  // the table entry of this wave's 16 positions of unit j
  auto entry = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, min(j, u1 - 1)) + 16 * wave;
    return table[min(p >> a.page_shift, a.max_pages - 1)];
  };
  // this wave's 16 rows of K and V of unit j to buffer j & 1. (Inline asm: through the
  // compiler's builtin, later LDS reads would wait for every load in flight.)
  // Whether there is no page.
  auto load = [&](int j, int e) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, j) + 16 * wave;
    const int page = paged_page(__builtin_amdgcn_readfirstlane(e), a.num_pages);
    if (lane == 0) lds.bad[j & 1][wave] = page < 0 ? 1 : 0;
    const size_t at = ((((size_t)max(page, 0) * a.plan.kv_heads + t.kv_head) << a.page_shift) + (p & page_mask)) * kRow;
    const uint64_t kb = (uint64_t)(uintptr_t)a.k + at, vb = (uint64_t)(uintptr_t)a.v + at;
    const uint32_t to = (j & 1) * kBuffer + wave * kWave;
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
      asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(k_off[u]), "s"(kb), "{m0}"(k_lds + to + u * 1024) : "memory");
      asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(v_off[u]), "s"(vb), "{m0}"(v_lds + to + u * 1024) : "memory");
    }
    return page < 0;
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16 acc[kDB];
#pragma unroll
  for (int db = 0; db < kDB; db++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[db][i] = 0.0f;

  __syncthreads();  // the last tile's LDS reads are done
  int entries = 0;
  bool none = false, none_next = false;  // this wave's 16 positions have no page
  if (u0 < u1) {
    none = load(u0, entry(u0));
    entries = entry(u0 + 1);
  }
  const int ti = (lane >> 2) & 3, tq = lane & 3, side = (lane >> 4) & 1;
  int v_at[kDB];  // (swz_v repeats every 4 rows, swz_k every 16)
#pragma unroll
  for (int db = 0; db < kDB; db++) {
    const int r = 4 * h + ti, c = 4 * db + 2 * side + (tq >> 1);
    v_at[db] = r * kRow + ((c ^ swz_v(r)) * 16) + (tq & 1) * 8;
  }
  int k_at[kKK];
#pragma unroll
  for (int kk = 0; kk < kKK; kk++) k_at[kk] = n32 * kRow + (((2 * kk + h) ^ swz_k(n32)) * 16);
  for (int j = u0; j < u1; j++, none = none_next) {
    const int p0 = span_position(s, kLargeUnit, j), buf = j & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // what no row sees: zeros in V
    if (none || p0 + 16 * wave + 16 > s.hi ||
        (a.plan.window > 0 && p0 + 16 * wave < s.lo && p0 + 16 * wave + 16 > s.sinks)) {
#pragma unroll
      for (int u = 0; u < kLoads; u++) {
        const int r = u * kLoadRows + lane / kChunks;
        if (none || !tile_sees(a, s, p0 + 16 * wave + r))
          *reinterpret_cast<u32x4 *>(&lds.v[buf][wave * kWave + u * 1024 + lane * 16]) = u32x4{0, 0, 0, 0};
      }
    }
    lds_barrier();
    if (j + 1 < u1) {
      none_next = load(j + 1, entries);
      entries = entry(j + 2);
    }
    const bool skip = !active || p0 > pos_hi ||
                      (a.plan.window > 0 && p0 + kLargeUnit <= pos_lo - a.plan.window + 1 && p0 >= s.sinks);
    if (skip) continue;
    // all K fragments requested before the first product, V's first half before the
    // softmax and its second half before the products of the first: the compiler
    // left to itself reads each just before its use
    Vec kf[2][kKK];
    const u32x4 bad4 = *reinterpret_cast<const u32x4 *>(lds.bad[buf]);
#pragma unroll
    for (int kk = 0; kk < kKK; kk++)
#pragma unroll
      for (int sb = 0; sb < 2; sb++)
        kf[sb][kk] = *reinterpret_cast<const Vec *>(&lds.k[buf][k_at[kk] + 32 * sb * kRow]);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 sc[2];
#pragma unroll
    for (int sb = 0; sb < 2; sb++)
#pragma unroll
      for (int i = 0; i < 16; i++) sc[sb][i] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < kKK; kk++)
#pragma unroll
      for (int sb = 0; sb < 2; sb++) sc[sb] = T::mfma32(kf[sb][kk], q[kk], sc[sb]);
    __builtin_amdgcn_sched_barrier(0);
    s16x4 vh[4][kDB][2];
    auto read_v = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < kDB; db++)
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++)
          vh[ks][db][q2] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (SH_PAGED_LDS s16x4 *)((SH_PAGED_LDS uint8_t *)lds.v[buf] + v_at[db] + (16 * ks + 8 * q2) * kRow));
    };
    read_v(0);
    read_v(1);
    __builtin_amdgcn_sched_barrier(0);
    const unsigned bad = __builtin_amdgcn_readfirstlane(bad4.x | (bad4.y << 1) | (bad4.z << 2) | (bad4.w << 3));
    const bool plain = bad == 0 && p0 + kLargeUnit <= pos_lo + 1 &&
                       (a.plan.window == 0 || p0 > pos_hi - a.plan.window || p0 + kLargeUnit <= s.sinks);
    if (!plain) {
#pragma unroll
      for (int sb = 0; sb < 2; sb++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int key = 32 * sb + 8 * (i / 4) + 4 * h + i % 4;
          if (((bad >> (2 * sb + i / 8)) & 1) || !sees(a, s, my_pos, p0 + key)) sc[sb][i] = -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < 2; sb++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, sc[sb][i]);
    mx = half_max(mx) * a.scale_log2;
    // the sums are rescaled only once a row's maximum has grown by 2^kSlack: until
    // then its weights are up to 2^kSlack times as large
    if (__any(mx > m_run + kSlack)) {
      const float m = fmaxf(m_run, mx);
      const float corr = m_run == m ? 1.0f : exp2_weight(m_run - m);
      m_run = m;
      l_run *= corr;
#pragma unroll
      for (int db = 0; db < kDB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[db][i] *= corr;
    }
    // (a row that has seen nothing yet: its weights are exp2(-infinity))
    const float off = (m_run == -INFINITY ? 0.0f : m_run) - T::kWeightLog2;
    float ls = 0.0f;
    Vec p[4];
#pragma unroll
    for (int sb = 0; sb < 2; sb++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float w = exp2_weight(fmaf(sc[sb][i], a.scale_log2, -off));
        p[2 * sb + i / 8][i % 8] = (Value)w;
        ls += w;
      }
    l_run += ls;
    __builtin_amdgcn_sched_barrier(0);
    read_v(2);
    read_v(3);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
#pragma unroll
      for (int db = 0; db < kDB; db++) {
        const Vec vf = __builtin_bit_cast(
            Vec, __builtin_shufflevector(vh[ks][db][0], vh[ks][db][1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[db] = T::mfma32(vf, p[ks], acc[db]);
      }
  }
  l_run += __shfl_xor(l_run, 32, 64);
  bool finite = true;
  if (32 * wave + n32 < rows) {
    finite = l_run < INFINITY;
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
    uint16_t *op = a.out + head_row(a, t.seq.row0 + s.first, t.kv_head, row) * kD;
    float *sp = slot_row<kD>(a, max(slot, 0), row);
#pragma unroll
    for (int db = 0; db < kDB; db++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const f32x4 x = {acc[db][4 * i], acc[db][4 * i + 1], acc[db][4 * i + 2], acc[db][4 * i + 3]};
        const int dim = 32 * db + 8 * i + 4 * h;
#pragma unroll
        for (int e = 0; e < 4; e++) finite = finite && __builtin_fabsf(x[e]) < INFINITY;
        if (slot < 0) {
          const Quad o = {(Value)(x[0] * inv), (Value)(x[1] * inv), (Value)(x[2] * inv), (Value)(x[3] * inv)};
          *reinterpret_cast<Quad *>(op + dim) = o;
        } else {
          *reinterpret_cast<f32x4 *>(sp + dim) = x;
        }
      }
    if (slot >= 0 && h == 0) {
      sp[kD] = m_run;
      sp[kD + 1] = l_run;
    }
  }
  return !__syncthreads_or(finite ? 0 : 1);
}

template <class T, int kD>
__global__ __launch_bounds__(kT, 2) void paged_large_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) LargeLds<kD> lds;
  __shared__ PlanLds plan;
  // consecutive pieces to one XCD: they share K and V
  const int worker = (blockIdx.x & 7) * (a.plan.workers >> 3) + (blockIdx.x >> 3);
  work_piece<kLargeMergeRows>(a, worker, plan, [&](const PieceStep &st) { return attn_large<T, kD>(a, st.tile, st.span, st.u0, st.u1, st.slot, lds); });
}

// ---- the merge ---------------------------------------------------------------------------
//
// out = sum_j 2^(m_j - M) acc_j / sum_j 2^(m_j - M) l_j, M = max_j m_j, over the
// parts j of a cut tile. The rows of all cut tiles are numbered through, in groups of
// kRows (a prefix sum over the workers' items), and a group taken by kWaves waves:
// one wave for 8 rows of large tiles, which have two or three parts, eight for a row
// of small ones, whose parts may be spread over all workers (of 8 times kWaves parts
// all loads are requested at once).
// Tiles with a part that is not finite are left to workgroup w of the first such
// worker w, which works them out in fp32, and its whole tiles too.
struct MergeLds {
  union {
    int prefix[kT + 1];
    PlanLds plan;
  };
  int waves[kMaxT / 64];
};

template <class T, int kD, int kThreads, int kWaves, int kRows>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnArgs a) {
  constexpr int kStep = 8 / kRows, kDims = kD / 64;
  typedef float Dims __attribute__((ext_vector_type(kDims)));
  __shared__ MergeLds lds;
  __shared__ Dims num_part[kWaves][64];
  __shared__ float top_part[kWaves], den_part[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // threads of two workers each
  static_assert(kSmallWorkers <= 2 * kT && kLargeWorkers <= 2 * kT, "two items per thread");
  const int workers = a.plan.workers;
  int sum = 0;
  if (tid < kT)
    for (int w = 2 * tid; w < min(2 * tid + 2, workers); w++) sum += a.groups[w];
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int o = __shfl_up(sum, off, 64);
    if (lane >= off) sum += o;
  }
  if (lane == 63) lds.waves[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; w++) sum += lds.waves[w];
  if (tid < kT) lds.prefix[tid + 1] = sum;
  if (tid == 0) lds.prefix[0] = 0;
  __syncthreads();
  const int total = lds.prefix[kT];
  constexpr int kAtOnce = kThreads / 64 / kWaves;
  for (int unit = blockIdx.x * kAtOnce + (kAtOnce > 1 ? wave / kWaves : 0); unit < total; unit += gridDim.x * kAtOnce) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kT / 64; i++) n += __popcll(__ballot(lds.prefix[1 + i * 64 + lane] <= unit));
    n = __builtin_amdgcn_readfirstlane(n);
    int g = unit - lds.prefix[n], w = 2 * n;
    if (g >= a.groups[w]) g -= a.groups[w++];
    const MergeItem it = a.items[w];
    const int r0 = g * kRows, rows = it.tokens * a.group;
    const int part0 = kWaves == 1 ? 0 : wave;
    float top[kRows], den[kRows];
    Dims num[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      top[i] = -INFINITY;
      den[i] = 0.0f;
      num[i] = 0.0f;
    }
    bool redo = false;
    for (int j0 = part0; j0 < it.parts; j0 += kWaves * kStep) {
      Dims x[kRows][kStep];
      float m[kRows][kStep], l[kRows][kStep];
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        const int j = min(j0 + kWaves * u, it.parts - 1), slot = j == 0 ? it.first_slot : 2 * (it.first_worker + j);
#pragma unroll
        for (int i = 0; i < kRows; i++) {
          const float *p = slot_row<kD>(a, slot, min(r0 + i, rows - 1));
          x[i][u] = *reinterpret_cast<const Dims *>(p + lane * kDims);
          m[i][u] = p[kD];
          l[i][u] = p[kD + 1];
        }
        redo = redo || a.redo[it.first_worker + j] != 0;
      }
#pragma unroll
      for (int i = 0; i < kRows; i++) {
        float t = top[i];
#pragma unroll
        for (int u = 0; u < kStep; u++)
          if (j0 + kWaves * u < it.parts) t = fmaxf(t, m[i][u]);
        const float c = t == top[i] ? 1.0f : exp2_weight(top[i] - t);
        top[i] = t;
        num[i] *= c;
        den[i] *= c;
#pragma unroll
        for (int u = 0; u < kStep; u++) {
          const float f = m[i][u] == -INFINITY || j0 + kWaves * u >= it.parts ? 0.0f : exp2_weight(m[i][u] - t);
          num[i] += f * x[i][u];
          den[i] = fmaf(f, l[i][u], den[i]);
        }
      }
    }
    if constexpr (kWaves > 1) {
      static_assert(kRows == 1, "the waves' sums are of one row");
      num_part[wave][lane] = num[0];
      if (lane == 0) {
        top_part[wave] = top[0];
        den_part[wave] = den[0];
      }
      redo = __syncthreads_or(redo ? 1 : 0);
      float t = top_part[0];
#pragma unroll
      for (int w2 = 1; w2 < kWaves; w2++) t = fmaxf(t, top_part[w2]);
      num[0] = 0.0f;
      den[0] = 0.0f;
#pragma unroll
      for (int w2 = 0; w2 < kWaves; w2++) {
        const float f = top_part[w2] == -INFINITY ? 0.0f : exp2_weight(top_part[w2] - t);
        num[0] += f * num_part[w2][lane];
        den[0] = fmaf(f, den_part[w2], den[0]);
      }
      __syncthreads();
    }
    if (redo || (kWaves > 1 && wave != 0)) continue;
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      if (r0 + i >= rows) break;
      const float inv = den[i] == 0.0f ? 0.0f : 1.0f / den[i];
      typename T::Value *o =
          reinterpret_cast<typename T::Value *>(a.out) + head_row(a, it.row0, it.kv_head, r0 + i) * kD + lane * kDims;
#pragma unroll
      for (int e = 0; e < kDims; e++) o[e] = (typename T::Value)(num[i][e] * inv);
    }
  }

  for (int w = blockIdx.x; w < workers; w += gridDim.x) {
    if (a.redo[w] == 0) continue;
    __syncthreads();  // lds.prefix is read
    MergeItem unused;
    long long piece;
    walk_piece(a.plan, w, lds.plan, &unused, &piece, [&](const PieceStep &st) {
      if (st.slot >= 0)  // a cut tile is the first flagged worker's
        for (int j = plan_first(st.tile, w, piece, w * piece); j < w; j++)
          if (a.redo[j] != 0) return true;
      attn_exact<T, kD>(a, st.tile, st.span);
      return true;
    });
    __syncthreads();
  }
}

// ---- the entry points ---------------------------------------------------------------

// Small tiles where every sequence's new tokens fit one.
bool small_tiles(int group, int max_new) { return group <= kSmallRows && (long long)group * max_new <= kSmallRows; }

size_t workspace_of(const sh_paged_kv *kv, int heads, int max_new) {
  const bool small = small_tiles(heads / kv->kv_heads, max_new);
  const size_t workers = small ? kSmallWorkers : kLargeWorkers, rows = small ? kSmallRows : kLargeRows;
  return workers * (sizeof(MergeItem) + 2 * sizeof(int)) + 2 * workers * rows * (kv->head_dim + 4) * 4;
}

int check_attn_sizes(const sh_paged_kv *kv, int tokens, int heads, int max_new) {
  if (const char *wrong = check_paged_sizes(kv, tokens, heads)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (!paged_dim_built(kv->head_dim))
    return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", kv->head_dim);
  if (max_new < 0) return fail(SH_ERR_INVALID_ARGUMENT, "max_new must not be negative");
  return SH_OK;
}

template <class T, int kD>
void launch(hipStream_t st, const PagedAttnArgs &a, bool small) {
  if (small) {
    paged_small_kernel<T, kD><<<a.plan.workers, kT, 0, st>>>(a);
    paged_merge_kernel<T, kD, 512, 8, kSmallMergeRows><<<a.plan.workers, 512, 0, st>>>(a);
  } else {
    paged_large_kernel<T, kD><<<a.plan.workers, kT, 0, st>>>(a);
    paged_merge_kernel<T, kD, kT, 1, kLargeMergeRows><<<a.plan.workers, kT, 0, st>>>(a);
  }
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
  const size_t bytes = (size_t)tokens * heads * kv->head_dim * 2, need = workspace_of(kv, heads, max_new);
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
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.max_pages = kv->max_pages;
  a.num_pages = kv->num_pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  const bool small = small_tiles(a.group, max_new);
  a.tile_rows = small ? kSmallRows : kLargeRows;
  a.scale_log2 = scale * 1.44269504f;
  PagedPlan &p = a.plan;
  p.starts = kv->starts;
  p.lengths = kv->lengths;
  p.batch = kv->batch;
  p.tokens = tokens;
  p.kv_heads = kv->kv_heads;
  p.capacity = kv->max_pages * kv->page_size;
  p.per_tile = a.tile_rows / a.group;
  p.unit = small ? 32 * 128 / kv->head_dim : kLargeUnit;
  p.unit_shift = __builtin_ctz((unsigned)p.unit);
  p.window = window;
  p.sinks = sinks;
  p.min_piece = small ? kSmallPiece : kLargePiece;
  p.workers = plan_workers(p.batch, p.kv_heads, tokens, p.capacity, p.per_tile, p.min_piece,
                           small ? kSmallWorkers : kLargeWorkers);
  p.inv_workers = std::nextafter(1.0 / p.workers, 2.0);
  a.items = static_cast<MergeItem *>(workspace);
  a.groups = reinterpret_cast<int *>(a.items + p.workers);
  a.redo = a.groups + p.workers;
  a.slots = reinterpret_cast<float *>(a.redo + p.workers);
  p.whole_below = small ? kSmallWhole : kLargeWhole;
  const hipStream_t st = stream_of(ctx);
  if (kv->head_dim == 64)
    launch<T, 64>(st, a, small);
  else
    launch<T, 128>(st, a, small);
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
  *bytes = workspace_of(kv, heads, max_new);
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
