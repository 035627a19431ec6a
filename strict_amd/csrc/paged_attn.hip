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
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define SH_PAGED_LDS __attribute__((address_space(3)))

// Pieces of a call, and the shortest, in positions: three workgroups per CU are
// resident with the small tiles, two with the large ones.
constexpr int kSmallRows = 16, kSmallWorkers = 768, kSmallPiece = 256;
constexpr int kLargeRows = 128, kLargeWorkers = 512, kLargePiece = 512;

struct PagedAttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int *table;
  PagedPlan plan;
  MergeItem *items;  // [workers]
  float *slots;      // [2 workers][rows of a tile][d + 4]
  int heads, group, max_pages, num_pages, page_shift, tile_rows;
  float scale_log2;
};

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
__device__ __forceinline__ void attn_small(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s, int u0,
                                           int u1, int slot, SmallLds<T, kD> &lds) {
  typedef typename T::Vec Vec;
  typedef typename T::Value Value;
  constexpr int kUnit = kSmallUnit<kD>, kBlocks = kUnit / 16, kKK = kD / 32, kDT = kD / 16;
  constexpr int kRow = kD * 2, kChunks = kD / 8, kVLoads = kUnit * kChunks / 64, kVRows = 64 / kChunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, grp = lane >> 4, rows = s.count * a.group;
  const int row = min(r16, rows - 1), my_pos = s.pos0 + row / a.group;
  const uint16_t *qp = a.q + ((size_t)(t.seq.row0 + s.first + row / a.group) * a.heads + t.kv_head * a.group +
                              row % a.group) * kD + grp * 8;
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
#pragma unroll
    for (int u = 0; u < kVLoads; u++) {
      const int r = u * kVRows + lane / kChunks, c = lane % kChunks;
      if (!plain && (((bad >> (u * kVRows / 16)) & 1) || !tile_sees(a, s, p0 + r))) vr[u] = u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4 *>(vl + r * kRow + ((c ^ swz(r)) * 16)) = vr[u];
    }
    if (next < u1) {
      __builtin_amdgcn_sched_barrier(0);
      load_v();
      *entries = entry(next + 4);
      __builtin_amdgcn_sched_barrier(0);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        sc[tt][e] *= a.scale_log2;
        if (!plain && (((bad >> tt) & 1) || !sees(a, s, my_pos, p0 + 16 * tt + 4 * grp + e))) sc[tt][e] = -INFINITY;
        mx = fmaxf(mx, sc[tt][e]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float m = fmaxf(m_run, mx);
    const float corr = m_run == m ? 1.0f : exp2_weight(m_run - m);
    m_run = m;
    float ls = 0.0f;
    Vec p[kBlocks / 2];
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float w = !plain && sc[tt][e] == -INFINITY ? 0.0f : exp2_weight(sc[tt][e] - (m - T::kWeightLog2));
        p[tt / 2][(tt & 1) * 4 + e] = (Value)w;
        ls += w;
      }
    l_run = l_run * corr + ls;  // this lane's positions; the groups are summed at the end
#pragma unroll
    for (int dt = 0; dt < kDT; dt++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[dt][e] *= corr;
    wait_lds();  // this wave's V rows are in LDS
    const int ti = (lane >> 2) & 3, tq = lane & 3;
#pragma unroll
    for (int sl = 0; sl < kBlocks / 2; sl++)
#pragma unroll
      for (int dt = 0; dt < kDT; dt++) {
        s16x4 half[2];
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++) {
          const int r = 32 * sl + 16 * q2 + 4 * grp + ti, c = 2 * dt + (tq >> 1);
          half[q2] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SH_PAGED_LDS s16x4 *)(
              (SH_PAGED_LDS uint8_t *)vl + r * kRow + ((c ^ swz(r)) * 16) + (tq & 1) * 8));
        }
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
  if (__syncthreads_or(finite ? 0 : 1)) {
    attn_exact<T, kD>(a, t, s, u0, u1, slot);
    __syncthreads();
  }
}

template <class T, int kD>
__global__ __launch_bounds__(kT, 3) void paged_small_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) SmallLds<T, kD> lds;
  walk_piece(a, blockIdx.x, [&](const PagedTile &t, const TileSpan &s, int u0, int u1, int slot) {
    attn_small<T, kD>(a, t, s, u0, u1, slot, lds);
  });
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

template <int kD>
struct LargeLds {
  uint8_t k[2][kLargeUnit * kD * 2], v[2][kLargeUnit * kD * 2];
  unsigned bad[2][4];  // a 16-position block without a page
};

template <class T, int kD>
__device__ __forceinline__ void attn_large(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s, int u0,
                                           int u1, int slot, LargeLds<kD> &lds) {
  typedef typename T::Vec Vec;
  typedef typename T::Value Value;
  typedef Value Quad __attribute__((ext_vector_type(4)));
  constexpr int kRow = kD * 2, kChunks = kD / 8, kKK = kD / 16, kDB = kD / 32;
  constexpr int kLoadRows = 64 / kChunks, kLoads = 16 / kLoadRows;  // of a wave's 16 positions
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5, rows = s.count * a.group;
  const bool active = 32 * wave < rows;  // (of the wave)
  const int row = min(32 * wave + n32, rows - 1), my_pos = s.pos0 + row / a.group;
  const int pos_lo = s.pos0 + min(32 * wave, rows - 1) / a.group, pos_hi = s.pos0 + min(32 * wave + 31, rows - 1) / a.group;
  const int *table = a.table + (size_t)t.b * a.max_pages;
  const int page_mask = (1 << a.page_shift) - 1;
  const uint16_t *qp = a.q + ((size_t)(t.seq.row0 + s.first + row / a.group) * a.heads + t.kv_head * a.group +
                              row % a.group) * kD + h * 8;
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
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16 acc[kDB];
#pragma unroll
  for (int db = 0; db < kDB; db++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[db][i] = 0.0f;

  __syncthreads();  // the last tile's LDS reads are done
  int entries = 0;
  if (u0 < u1) {
    load(u0, entry(u0));
    entries = entry(u0 + 1);
  }
  for (int j = u0; j < u1; j++) {
    const int p0 = span_position(s, kLargeUnit, j), buf = j & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // what no row sees: zeros in V
    if (__builtin_amdgcn_readfirstlane((int)lds.bad[buf][wave]) || p0 + 16 * wave + 16 > s.hi ||
        (a.plan.window > 0 && p0 + 16 * wave < s.lo && p0 + 16 * wave + 16 > s.sinks)) {
      const bool none = lds.bad[buf][wave] != 0;
#pragma unroll
      for (int u = 0; u < kLoads; u++) {
        const int r = u * kLoadRows + lane / kChunks;
        if (none || !tile_sees(a, s, p0 + 16 * wave + r))
          *reinterpret_cast<u32x4 *>(&lds.v[buf][wave * kWave + u * 1024 + lane * 16]) = u32x4{0, 0, 0, 0};
      }
    }
    lds_barrier();
    if (j + 1 < u1) {
      load(j + 1, entries);
      entries = entry(j + 2);
    }
    const bool skip = !active || p0 > pos_hi ||
                      (a.plan.window > 0 && p0 + kLargeUnit <= pos_lo - a.plan.window + 1 && p0 >= s.sinks);
    if (skip) continue;
    const unsigned bad0 = lds.bad[buf][0], bad1 = lds.bad[buf][1], bad2 = lds.bad[buf][2], bad3 = lds.bad[buf][3];
    const unsigned bad = __builtin_amdgcn_readfirstlane(bad0 | (bad1 << 1) | (bad2 << 2) | (bad3 << 3));
    const bool plain = bad == 0 && p0 + kLargeUnit <= pos_lo + 1 &&
                       (a.plan.window == 0 || p0 > pos_hi - a.plan.window || p0 + kLargeUnit <= s.sinks);
    f32x16 sc[2];
#pragma unroll
    for (int sb = 0; sb < 2; sb++) {
#pragma unroll
      for (int i = 0; i < 16; i++) sc[sb][i] = 0.0f;
      const int r = 32 * sb + n32;
#pragma unroll
      for (int kk = 0; kk < kKK; kk++) {
        const Vec kf = *reinterpret_cast<const Vec *>(&lds.k[buf][r * kRow + (((2 * kk + h) ^ swz_k(r)) * 16)]);
        sc[sb] = T::mfma32(kf, q[kk], sc[sb]);
      }
    }
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
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2;
    if (__any(mx > m_run)) {
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
    const int ti = (lane >> 2) & 3, tq = lane & 3, side = (lane >> 4) & 1;
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
#pragma unroll
      for (int db = 0; db < kDB; db++) {
        s16x4 half[2];
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++) {
          const int r = 16 * ks + 8 * q2 + 4 * h + ti, c = 4 * db + 2 * side + (tq >> 1);
          half[q2] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SH_PAGED_LDS s16x4 *)(
              (SH_PAGED_LDS uint8_t *)lds.v[buf] + r * kRow + ((c ^ swz_v(r)) * 16) + (tq & 1) * 8));
        }
        const Vec vf = __builtin_bit_cast(Vec, __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[db] = T::mfma32(vf, p[ks], acc[db]);
      }
  }
  l_run += __shfl_xor(l_run, 32, 64);
  bool finite = true;
  if (32 * wave + n32 < rows) {
    finite = l_run < INFINITY;
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
    uint16_t *op = a.out + ((size_t)(t.seq.row0 + s.first + row / a.group) * a.heads + t.kv_head * a.group +
                            row % a.group) * kD;
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
  if (__syncthreads_or(finite ? 0 : 1)) attn_exact<T, kD>(a, t, s, u0, u1, slot);
}

template <class T, int kD>
__global__ __launch_bounds__(kT, 2) void paged_large_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) LargeLds<kD> lds;
  // consecutive pieces to one XCD: they share K and V
  const int worker = (blockIdx.x & 7) * (kLargeWorkers / 8) + (blockIdx.x >> 3);
  walk_piece(a, worker, [&](const PagedTile &t, const TileSpan &s, int u0, int u1, int slot) {
    attn_large<T, kD>(a, t, s, u0, u1, slot, lds);
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

// Small tiles where every sequence's new tokens fit one.
bool small_tiles(int group, int max_new) { return group <= kSmallRows && (long long)group * max_new <= kSmallRows; }

size_t workspace_of(const sh_paged_kv *kv, int heads, int max_new) {
  const bool small = small_tiles(heads / kv->kv_heads, max_new);
  const size_t workers = small ? kSmallWorkers : kLargeWorkers, rows = small ? kSmallRows : kLargeRows;
  return workers * sizeof(MergeItem) + 2 * workers * rows * (kv->head_dim + 4) * 4;
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
  a.max_pages = kv->max_pages;
  a.num_pages = kv->num_pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  const bool small = small_tiles(a.group, max_new);
  const int workers = small ? kSmallWorkers : kLargeWorkers;
  a.tile_rows = small ? kSmallRows : kLargeRows;
  a.scale_log2 = scale * 1.44269504f;
  a.items = static_cast<MergeItem *>(workspace);
  a.slots = reinterpret_cast<float *>(a.items + workers);
  PagedPlan &p = a.plan;
  p.starts = kv->starts;
  p.lengths = kv->lengths;
  p.batch = kv->batch;
  p.tokens = tokens;
  p.kv_heads = kv->kv_heads;
  p.capacity = kv->max_pages * kv->page_size;
  p.per_tile = a.tile_rows / a.group;
  p.unit = small ? 32 * 128 / kv->head_dim : kLargeUnit;
  p.window = window;
  p.sinks = sinks;
  p.workers = workers;
  p.min_piece = small ? kSmallPiece : kLargePiece;
  p.whole_below = 0;
  const hipStream_t st = stream_of(ctx);
  if (kv->head_dim == 64) {
    if (small)
      paged_small_kernel<T, 64><<<workers, kT, 0, st>>>(a);
    else
      paged_large_kernel<T, 64><<<workers, kT, 0, st>>>(a);
    paged_merge_kernel<T, 64><<<workers, kT, 0, st>>>(a);
  } else {
    if (small)
      paged_small_kernel<T, 128><<<workers, kT, 0, st>>>(a);
    else
      paged_large_kernel<T, 128><<<workers, kT, 0, st>>>(a);
    paged_merge_kernel<T, 128><<<workers, kT, 0, st>>>(a);
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
