// What the attention kernels over pages of either kind share (paged_attn.hip, 16-bit
// values; paged_attn8.hip, 8-bit values with scales): how a workgroup walks its piece of
// a call, the sums' places, the merge of cut tiles, and the tiles that the matrix
// products cannot do.
//
// A call is divided into equal pieces of work (paged.h): workgroup w takes the
// tiles of its piece, a tile being some tokens of one sequence with the query
// heads of one KV head, its rows (token, head) numbered token * G + head. A tile
// that lies in one piece is written to the output; one cut between pieces leaves
// a part in each of its workgroups' slots (V sums, maximum and sum of weights
// per row), and a second kernel merges the parts. That kernel also works out again,
// in fp32 without matrix products, what came out not finite (infinities and NaN in
// q, K or V, or in places of V that only some of a tile's rows see), sums beyond kMaxSum
// and rows whose largest score is beyond kMaxScore.
//
// Softmax runs over the positions in order with a running maximum, in base 2:
// s = q.k scale log2(e), weights 2^(s - max) (times 2^7 in fp16). The weights are
// rounded to 16 bits for the product with V (whose matrix instructions take both
// operands so; those of fp32 run at a sixteenth of the rate): 8,192 bf16 tokens are then
// off by 2.2e-3 of their size where the rounding of the results alone makes 1.6e-3.
// Their sum is that of the rounded ones: what the roundings of many equal weights have
// in common goes out with the division.
#pragma once

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

// How a call is divided: rows of a tile, pieces at most (as many as workgroups are
// resident), the shortest piece and the tiles that are not cut, in positions. (One
// token over 777 positions 14.2 us a call; with shortest pieces of twice and four times
// that 15.0 and 16.1. 8 sequences of up to 200 tokens of 12 heads of 64: 28.0, 29.6 and
// 37.5. Tiles left whole up to half or twice as many positions: within 5 % either way.)
struct Variant {
  int rows, workers, min_piece, whole_below;
};
constexpr Variant kSmall = {16, 512, 64, 192}, kLarge = {128, 512, 128, 256};
constexpr int kMaxWorkers = 512;
constexpr int kLargeUnit = 64;  // positions of a large tile's unit

struct PagedAttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int *table;
  PagedPlan plan;
  MergeItem *items;  // [workers]
  int *groups;       // [workers]: rows to merge of the worker's item, in groups
  int *redo;         // [workers]: 1: some of the worker's results are to be worked out again
  float *slots;      // [2 workers][rows of a tile * (d + 2)]
  int heads, group, group_inv, max_pages, num_pages, page_shift, tile_rows;
  float scale_log2;
  float no_score;    // a row's maximum that says it has no scores: -infinity or NaN (none)
};

// Token of a tile's row (r <= 255, group <= 128: exact), and its row of heads in q
// and out.
__device__ __forceinline__ int token_of(const PagedAttnArgs &a, int r) { return (r * a.group_inv) >> 16; }
__device__ __forceinline__ size_t head_row(const PagedAttnArgs &a, int row0, int kv_head, int r) {
  const int token = token_of(a, r);
  return (size_t)(row0 + token) * a.heads + kv_head * a.group + (r - token * a.group);
}

// A slot: the V sums, then every row's maximum and sum of weights. The V sums of
// small tiles lie row by row, those of large ones as the lanes hold them (4 values
// per lane, a KiB at once): written row by row, 16 bytes a row, they took as long as
// six units.
template <int kD>
__device__ __forceinline__ float *slot_of(const PagedAttnArgs &a, int slot) {
  return a.slots + (size_t)slot * a.tile_rows * (kD + 2);
}
template <int kD>
__device__ __forceinline__ float *slot_stats(const PagedAttnArgs &a, int slot, int r) {
  return slot_of<kD>(a, slot) + a.tile_rows * kD + 2 * r;
}
// Values 4 i .. 4 i + 3 of block db of the wave's accumulators.
template <int kD>
__device__ __forceinline__ f32x4 *slot_large(const PagedAttnArgs &a, int slot, int wave, int db, int i) {
  return reinterpret_cast<f32x4 *>(slot_of<kD>(a, slot)) + ((wave * (kD / 32) + db) * 4 + i) * 64 + (threadIdx.x & 63);
}

// Where the results of a tile's part go: the output (slot -1) or a slot.
template <class T, int kD>
__device__ __forceinline__ void store_value(const PagedAttnArgs &a, const PagedTile &t, const TileSpan &s,
                                            int slot, int r, int dim, float acc, float l) {
  if (slot < 0) {
    const size_t row = head_row(a, t.seq.row0 + s.first, t.kv_head, r);
    reinterpret_cast<typename T::Value *>(a.out)[row * kD + dim] = (typename T::Value)(l == 0.0f ? 0.0f : acc / l);
  } else {
    slot_of<kD>(a, slot)[r * kD + dim] = acc;
  }
}

__device__ __forceinline__ float exp2_weight(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's maximum fits. -infinity is that of a row that sees nothing, or whose products
// are below fp32's range: with scales of up to 2^20 only those of q.k below -2^108. With
// larger ones a row of it is worked out again. (To ask what a row sees, where its sums are
// written, was 1 us of 35 for 8 sequences of up to 333 tokens, and so was a branch.)
constexpr float kPlainScale = 0x1p20f;
template <class T>
__device__ __forceinline__ bool score_fits(const PagedAttnArgs &a, float m) {
  return __builtin_fabsf(m) < T::kMaxScore || m == a.no_score;
}

// V sums that leave room for those of all parts (bf16 values of 2^64 and more reach it):
// beyond, the mean may be in fp32's range where the sums are not.
constexpr float kMaxSum = 0x1p100f;
__device__ __forceinline__ bool sum_fits(float x) { return __builtin_fabsf(x) < kMaxSum; }

// What a token at position `pos` sees of the positions from p on: i of them on if
// i <= last and (i >= first or i < sinks). (As limits of i, which the compiler has as
// constants: as positions it would keep all of them in registers.)
struct Sees {
  int last, first, sinks;
  __device__ __forceinline__ Sees(const PagedAttnArgs &a, const TileSpan &s, int pos, int p)
      : last(pos - p), first(a.plan.window == 0 ? -p : pos - a.plan.window + 1 - p), sinks(s.sinks - p) {}
  __device__ __forceinline__ bool operator()(int i) const { return i <= last && (i >= first || i < sinks); }
};

// Pages of 16-bit values as attn_exact reads them. (C of the templates below: this, or
// what stands for it of other pages.)
template <class T>
struct Pages16 {
  typedef T Type;
  typedef PagedAttnArgs Args;
  typedef long long Row;
  template <int kD>
  static __device__ __forceinline__ Row row(const Args &a, int page, int kv_head, int in_page) {
    return (((((long long)page * a.plan.kv_heads + kv_head) << a.page_shift) + in_page) * kD);
  }
  static __device__ __forceinline__ Row row_of_lane(Row r, int lane) { return __shfl(r, lane, 64); }
  static __device__ __forceinline__ float k(const Args &a, Row r, int c) {
    return (float)reinterpret_cast<const typename T::Value *>(a.k)[r + c];
  }
  static __device__ __forceinline__ float v(const Args &a, Row r, int c) {
    return (float)reinterpret_cast<const typename T::Value *>(a.v)[r + c];
  }
};

// A tile in fp32, a wave per row, a lane per position of 64: whatever the values are.
// The maximum is q.k's, the scale taken after it is subtracted, so that the largest
// weight is 1 however large the scores; the V sums are those of weights divided by their
// sum so far, and so no larger than the values. A score of -infinity, and a weight that
// is 0 in fp32, adds nothing. For tiles that the matrix products cannot do, and slow:
// each lane reads a row of K of its own, and a worker with one such tile has all of its
// tiles done again. A NaN that one of 48 decode rows of up to 4,352 positions sees:
// 0.11 -> 4.0 ms; one in the last of 8,192 tokens over 12,288 positions: 0.6 -> 285 ms.
template <class C, int kD>
__device__ void attn_exact(const typename C::Args &a, const PagedTile &t, const TileSpan &s) {
  typedef typename C::Type T;
  typedef typename T::Value Value;
  constexpr int kDims = kD / 64;
  const int lane = threadIdx.x & 63, rows = s.count * a.group;
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
        bool seen = p < end && Sees(a, s, pos, p)(0);
        typename C::Row at = {};  // the position's k and v
        if (seen) {
          const int page = paged_page(a.table[(size_t)t.b * a.max_pages + (p >> a.page_shift)], a.num_pages);
          seen = page >= 0;
          at = C::template row<kD>(a, max(page, 0), t.kv_head, p & ((1 << a.page_shift) - 1));
        }
        float dot = -INFINITY;
        if (seen) {
          dot = 0.0f;
          for (int c = 0; c < kD; c++) dot = fmaf((float)q[c], C::k(a, at, c), dot);
        }
        const float top = fmaxf(m, wave_max(dot));
        const float w = dot == -INFINITY ? 0.0f : exp2_weight((dot - top) * a.scale_log2);
        const float c = top == m ? 1.0f : exp2_weight((m - top) * a.scale_log2);
        const float before = l * c;
        l = before + wave_sum(w);
        m = top;
        const float kept = l == 0.0f ? 0.0f : before / l, part = l == 0.0f ? 0.0f : w / l;
#pragma unroll
        for (int j = 0; j < kDims; j++) acc[j] *= kept;
        for (int i = 0; i < 64; i++) {
          const float wi = __shfl(part, i, 64);
          const typename C::Row ai = C::row_of_lane(at, i);
          if (wi == 0.0f) continue;
#pragma unroll
          for (int j = 0; j < kDims; j++) acc[j] = fmaf(wi, C::v(a, ai, lane + 64 * j), acc[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kDims; j++) store_value<T, kD>(a, t, s, -1, r, lane + 64 * j, acc[j], 1.0f);
  }
}

// The line's division among the workers, in LDS.
struct PlanLds {
  Line prefix[kT + 1], waves[kMaxT / 64], largest[kMaxT / 64];
  PlanSeq seqs[kT];  // where a thread has one sequence
};

template <int kCtrl, int kRowMask>
__device__ __forceinline__ Line dpp_line(Line v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, kRowMask, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kCtrl, kRowMask, 0xf, false);
  return __builtin_bit_cast(Line, ((uint64_t)hi << 32) | lo);
}

// Sum (maximum) of lanes 0 .. own, by lane moves (row_shr:1, 2, 4, 8, row_bcast:15,
// 31; a lane that gets nothing gets 0): a fifth of the time of LDS permutes.
template <class Op>
__device__ __forceinline__ Line wave_scan_line(Line v, Op op) {
  v = op(v, dpp_line<0x111, 0xf>(v));
  v = op(v, dpp_line<0x112, 0xf>(v));
  v = op(v, dpp_line<0x114, 0xf>(v));
  v = op(v, dpp_line<0x118, 0xf>(v));
  v = op(v, dpp_line<0x142, 0xa>(v));
  v = op(v, dpp_line<0x143, 0xc>(v));
  return v;
}

// Prefix sums of the sequences' costs, by kT threads (of kT or more) of `per`
// sequences each, and the largest tile's cost per wave.
__device__ __forceinline__ void scan_costs(const PagedPlan &p, int per, PlanLds &lds) {
  const int t = threadIdx.x;
  Line sum = 0, largest = 0;
  for (int b = t * per; b < min((t + 1) * per, p.batch); b++) {
    const PlanSeq s = plan_sequence(p, b);
    if (per == 1) lds.seqs[t] = s;
    sum = plan_add(sum, s.one * p.kv_heads);
    largest = fmax(largest, plan_last(p, s));
  }
  sum = wave_scan_line(sum, [](Line x, Line y) { return plan_add(x, y); });
  largest = wave_scan_line(largest, [](Line x, Line y) { return fmax(x, y); });
  if ((t & 63) == 63) {
    lds.waves[t >> 6] = sum;
    lds.largest[t >> 6] = largest;
  }
  __syncthreads();
  for (int w = 0; w < (t >> 6); w++) sum = plan_add(sum, lds.waves[w]);
  if (t < kT) lds.prefix[t + 1] = sum;
  if (t == 0) lds.prefix[0] = 0;
  __syncthreads();
}

// A value that is the same in every lane, as the compiler cannot know of one from LDS.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ Line uniform(Line x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(Line, ((uint64_t)(uint32_t)uniform((int)(u >> 32)) << 32) | (uint32_t)uniform((int)u));
}

// The last i < kT with prefix[i] <= x: how many of the values from prefix[1] on are
// (a wave looks at all 256 at once).
__device__ __forceinline__ int find_part(const PlanLds &lds, Line x) {
  const int lane = threadIdx.x & 63;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; i++) n += __popcll(__ballot(lds.prefix[1 + i * 64 + lane] <= x));
  return min(n, kT - 1);
}

// The worker that a workgroup is, if workgroups of one XCD are to be consecutive
// workers, which share K and V. Of fewer pieces than workers each XCD takes an eighth
// (392 tiles on 512: 66.4 -> 64.0 us a call; 8 sequences of up to 200 tokens 28 -> 27).
__device__ __forceinline__ int worker_by_xcd(const PagedPlan &p, Line total, Line piece) {
  const int used = min((int)plan_div(total + piece - 1, piece), p.workers), per = (used + 7) >> 3;
  const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
  return i < per ? xcd * per + i : 8 * i + xcd;
}

// A worker's piece, step by step: part(step), which says whether its results are
// sound: finite, of sums and scores that fit. Returns whether all are. kByXcd: *worker is to be found.
template <bool kByXcd, class Part>
__device__ __forceinline__ bool walk_piece(const PagedPlan &p, int *worker, PlanLds &lds, MergeItem *item, Part part) {
  const int per = (p.batch + kT - 1) / kT;
  scan_costs(p, per, lds);
  Line largest = 0;
#pragma unroll
  for (int w = 0; w < kT / 64; w++) largest = fmax(largest, lds.largest[w]);
  const Line total = uniform(lds.prefix[kT]), piece = uniform(plan_piece(p, total, largest));
  const int me = kByXcd ? uniform(worker_by_xcd(p, total, piece)) : *worker;
  *worker = me;
  const Line x0 = me * piece, end = uniform(fmin(x0 + piece, total));
  bool sound = true;
  Line x = x0;
  while (uniform(x < end ? 1 : 0)) {
    const int i = uniform(find_part(lds, x)), b = plan_part_first(p, i, per);
    const PagedTile t = plan_locate(p, per == 1 ? lds.seqs[b] : plan_sequence(p, b), i, per, lds.prefix[i], x);
    PieceStep st = plan_step(p, t, piece, me, x0, x, item);
    for (int *v : {&st.tile.seq.row0, &st.tile.seq.n, &st.tile.seq.len, &st.tile.b, &st.tile.kv_head, &st.tile.tile,
                   &st.span.first, &st.span.count, &st.span.pos0, &st.span.lo, &st.span.hi, &st.span.sinks,
                   &st.span.units, &st.span.sink_units, &st.span.gap, &st.u0, &st.u1, &st.slot})
      *v = uniform(*v);
    st.run = uniform(st.run ? 1 : 0) != 0;
    st.more = uniform(st.more ? 1 : 0) != 0;
    x = uniform(t.begin + t.cost);
    if (!st.more) break;
    if (st.run && !part(st, piece)) sound = false;
  }
  return sound;
}

// A workgroup of the main kernels.
// kMergeRows: rows of an item's group, kMergeCols: groups that share rows.
template <bool kByXcd, int kMergeRows, int kMergeCols, class Part>
__device__ __forceinline__ void work_piece(const PagedAttnArgs &a, PlanLds &lds, Part part) {
  int worker = blockIdx.x;
  MergeItem item = {0, 0, 0, 0, 0, 0};
  const bool sound = walk_piece<kByXcd>(a.plan, &worker, lds, &item, part);
  if (threadIdx.x == 0) {
    a.items[worker] = item;
    a.groups[worker] = item.parts > 0 ? (item.tokens * a.group + kMergeRows - 1) / kMergeRows * kMergeCols : 0;
    a.redo[worker] = sound ? 0 : 1;
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

// x *= f where `really` is not 0 (the same in every lane), in place, x in the registers
// named. (Asm, with the branch inside: of a branch around the products the compiler
// keeps both versions of an accumulator and moves one to the other. The pauses are what
// a product's result and its next addend need, which the compiler does not add for asm.
// One branch for all of them: with one each, 8 sequences of up to 333 tokens took 35.3 us
// and not 34.9.)
#define SH_MUL1(r) "v_mul_f32 v" #r ", %[f], v" #r "\n\t"
#define SH_MUL4(a, b, c, d) SH_MUL1(a) SH_MUL1(b) SH_MUL1(c) SH_MUL1(d)
#define SH_SCALE_IF "s_cmp_eq_u32 %[really], 0\n\ts_cbranch_scc1 .Lpaged_scale%=\n\ts_nop 15\n\ts_nop 3\n\t"
#define SH_SCALE_END "s_nop 3\n.Lpaged_scale%=:"
#define SH_MUL_64_95                                                                                      \
  SH_MUL4(64, 65, 66, 67) SH_MUL4(68, 69, 70, 71) SH_MUL4(72, 73, 74, 75) SH_MUL4(76, 77, 78, 79)         \
  SH_MUL4(80, 81, 82, 83) SH_MUL4(84, 85, 86, 87) SH_MUL4(88, 89, 90, 91) SH_MUL4(92, 93, 94, 95)
#define SH_MUL_96_127                                                                                     \
  SH_MUL4(96, 97, 98, 99) SH_MUL4(100, 101, 102, 103) SH_MUL4(104, 105, 106, 107)                         \
  SH_MUL4(108, 109, 110, 111) SH_MUL4(112, 113, 114, 115) SH_MUL4(116, 117, 118, 119)                     \
  SH_MUL4(120, 121, 122, 123) SH_MUL4(124, 125, 126, 127)
__device__ __forceinline__ void scale_if(f32x16 (&x)[2], float f, int really) {
  asm volatile(SH_SCALE_IF SH_MUL_64_95 SH_SCALE_END
               : "+{v[64:79]}"(x[0]), "+{v[80:95]}"(x[1])
               : [f] "v"(f), [really] "s"(really)
               : "scc");
}
__device__ __forceinline__ void scale_if(f32x16 (&x)[4], float f, int really) {
  asm volatile(SH_SCALE_IF SH_MUL_64_95 SH_MUL_96_127 SH_SCALE_END
               : "+{v[64:79]}"(x[0]), "+{v[80:95]}"(x[1]), "+{v[96:111]}"(x[2]), "+{v[112:127]}"(x[3])
               : [f] "v"(f), [really] "s"(really)
               : "scc");
}

// ---- the merge ---------------------------------------------------------------------------
//
// out = sum_j 2^(m_j - M) acc_j / sum_j 2^(m_j - M) l_j, M = max_j m_j, over the
// parts j of a cut tile. The cut tiles' work is numbered through in groups (a prefix
// sum over the workers' items): of small tiles a row, whose parts, perhaps spread over
// all workers, are taken by 8 waves, 8 at once in each; of large tiles, of two or three
// parts mostly, 32 rows by 32 dims a wave, as the main kernel's lanes held them.
// Tiles with a part that is not sound are left to workgroup w of the first such
// worker w, which works them out in fp32, and its whole tiles too.
struct MergeLds {
  union {
    struct {
      int prefix[kT + 1], first[kT];  // of worker 2 i: the groups before its, and its groups
    };
    PlanLds plan;
  };
  int waves[kMaxT / 64];
};

// Group `unit`'s item, and which of its groups. False: there are fewer.
__device__ __forceinline__ bool find_item(const PagedAttnArgs &a, const MergeLds &lds, int unit, MergeItem *it, int *g) {
  const int lane = threadIdx.x & 63;
  if (unit >= uniform(lds.prefix[kT])) return false;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; i++) n += __popcll(__ballot(lds.prefix[1 + i * 64 + lane] <= unit));
  n = uniform(n);
  int w = 2 * n;
  *g = unit - uniform(lds.prefix[n]);
  const int first = uniform(lds.first[n]);
  if (*g >= first) {
    *g -= first;
    w++;
  }
  *it = a.items[w];
  return true;
}

// Prefix sums of the items' groups, by threads of two workers each.
__device__ __forceinline__ void scan_items(const PagedAttnArgs &a, MergeLds &lds) {
  static_assert(kMaxWorkers <= 2 * kT, "two items per thread");
  const int tid = threadIdx.x, wave = tid >> 6;
  int2 two = make_int2(0, 0);  // (workers are a multiple of 8)
  if (2 * tid < a.plan.workers) two = reinterpret_cast<const int2 *>(a.groups)[tid];
  int sum = two.x + two.y;
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xf, 0xf, false);  // (as in wave_scan_line)
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xf, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xf, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xf, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x142, 0xa, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x143, 0xc, 0xf, false);
  if ((tid & 63) == 63) lds.waves[wave] = sum;
  __syncthreads();
  if (tid < kT) {
#pragma unroll
    for (int w = 0; w < kT / 64; w++) sum += w < wave ? lds.waves[w] : 0;
    lds.prefix[tid + 1] = sum;
    lds.first[tid] = two.x;
  }
  if (tid == 0) lds.prefix[0] = 0;
  __syncthreads();
}

// The flagged workers' tiles.
template <class C, int kD>
__device__ __forceinline__ void redo_tiles(const typename C::Args &a, MergeLds &lds, int flagged) {
  int w = blockIdx.x;
  if (flagged == 0) return;
  __syncthreads();  // lds.prefix is read
  MergeItem unused;
  walk_piece<false>(a.plan, &w, lds.plan, &unused, [&](const PieceStep &st, Line piece) {
    if (st.slot >= 0)  // a cut tile is the first flagged worker's
      for (int j = plan_first(st.tile, w, piece, w * piece); j < w; j++)
        if (a.redo[j] != 0) return true;
    attn_exact<C, kD>(a, st.tile, st.span);
    return true;
  });
}

// (read at once, for the end; there are as many workgroups as workers, or more)
__device__ __forceinline__ int redo_flag(const PagedAttnArgs &a) {
  return (int)blockIdx.x < a.plan.workers ? a.redo[blockIdx.x] : 0;
}

__device__ __forceinline__ int part_slot(const MergeItem &it, int j) {
  return j == 0 ? it.first_slot : 2 * (it.first_worker + j);
}

constexpr int kMergeT = 512;
template <class C, int kD>
__global__ __launch_bounds__(kMergeT) void paged_merge_small_kernel(const typename C::Args a) {
  typedef typename C::Type T;
  constexpr int kWaves = kMergeT / 64, kStep = 8, kDims = kD / 64;
  typedef float Dims __attribute__((ext_vector_type(kDims)));
  __shared__ MergeLds lds;
  __shared__ Dims num_part[kWaves][64];
  __shared__ float top_part[kWaves], den_part[kWaves];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int flagged = redo_flag(a);
  scan_items(a, lds);
  MergeItem it;
  int r;
  for (int unit = blockIdx.x; find_item(a, lds, unit, &it, &r); unit += gridDim.x) {
    float top = -INFINITY, den = 0.0f;
    Dims num = 0.0f;
    bool redo = false;
    for (int j0 = wave; j0 < it.parts; j0 += kWaves * kStep) {
      Dims x[kStep];
      // (the maxima and sums of the wave's parts by a lane each; a load more for each
      // part, and for those that are not there, was 2 us of 9)
      const int mine = j0 + kWaves * lane;
      float my_m = -INFINITY, my_l = 0.0f;
      int again = 0;
      if (lane < kStep && mine < it.parts) {
        const f32x2 stat = *reinterpret_cast<const f32x2 *>(slot_stats<kD>(a, part_slot(it, mine), r));
        my_m = stat.x;
        my_l = stat.y;
        again = a.redo[it.first_worker + mine];
      }
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        x[u] = 0.0f;
        const int j = j0 + kWaves * u;
        if (j < it.parts)
          x[u] = *reinterpret_cast<const Dims *>(slot_of<kD>(a, part_slot(it, j)) + r * kD + lane * kDims);
      }
      redo = redo || __any(again != 0);
      float m[kStep], l[kStep], t = top;
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        m[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_m), u));
        l[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_l), u));
        t = fmaxf(t, m[u]);
      }
      const float c = t == top ? 1.0f : exp2_weight(top - t);
      top = t;
      num *= c;
      den *= c;
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        const float f = m[u] == -INFINITY ? 0.0f : exp2_weight(m[u] - t);
        num += f * x[u];
        den = fmaf(f, l[u], den);
      }
    }
    num_part[wave][lane] = num;
    if (lane == 0) {
      top_part[wave] = top;
      den_part[wave] = den;
    }
    redo = __syncthreads_or(redo ? 1 : 0);
    if (wave == 0 && !redo) {
      float t = top_part[0];
#pragma unroll
      for (int w = 1; w < kWaves; w++) t = fmaxf(t, top_part[w]);
      num = 0.0f;
      den = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float f = top_part[w] == -INFINITY ? 0.0f : exp2_weight(top_part[w] - t);
        num += f * num_part[w][lane];
        den = fmaf(f, den_part[w], den);
      }
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;
      typename T::Value *o =
          reinterpret_cast<typename T::Value *>(a.out) + head_row(a, it.row0, it.kv_head, r) * kD + lane * kDims;
#pragma unroll
      for (int e = 0; e < kDims; e++) o[e] = (typename T::Value)(num[e] * inv);
    }
    __syncthreads();  // the parts are read
  }
  redo_tiles<C, kD>(a, lds, flagged);
}

template <class C, int kD>
__global__ __launch_bounds__(kT) void paged_merge_large_kernel(const typename C::Args a) {
  typedef typename C::Type T;
  constexpr int kStep = 3, kDB = kD / 32;
  typedef typename T::Value Value;
  typedef Value Quad __attribute__((ext_vector_type(4)));
  __shared__ MergeLds lds;
  const int lane = threadIdx.x & 63, n32 = lane & 31, h = lane >> 5;
  const int flagged = redo_flag(a);
  scan_items(a, lds);
  MergeItem it;
  int g;
  for (int unit = blockIdx.x * (kT / 64) + uniform((int)threadIdx.x >> 6); find_item(a, lds, unit, &it, &g);
       unit += gridDim.x * (kT / 64)) {
    const int db = g % kDB, wave = g / kDB, rows = it.tokens * a.group, row = min(32 * wave + n32, rows - 1);
    float top = -INFINITY, den = 0.0f;
    f32x4 num[4];
#pragma unroll
    for (int i = 0; i < 4; i++) num[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool redo = false;
    for (int j0 = 0; j0 < it.parts; j0 += kStep) {
      f32x4 x[kStep][4];
      float m[kStep], l[kStep], t = top;
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        const int j = j0 + u, slot = part_slot(it, j);
        m[u] = -INFINITY;
        l[u] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) x[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (j < it.parts) {
          const f32x2 stat = *reinterpret_cast<const f32x2 *>(slot_stats<kD>(a, slot, row));
          m[u] = stat.x;
          l[u] = stat.y;
#pragma unroll
          for (int i = 0; i < 4; i++) x[u][i] = *slot_large<kD>(a, slot, wave, db, i);
          redo = redo || a.redo[it.first_worker + j] != 0;
        }
      }
#pragma unroll
      for (int u = 0; u < kStep; u++) t = fmaxf(t, m[u]);
      const float c = t == top ? 1.0f : exp2_weight(top - t);
      top = t;
      den *= c;
#pragma unroll
      for (int i = 0; i < 4; i++) num[i] *= c;
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        const float f = m[u] == -INFINITY ? 0.0f : exp2_weight(m[u] - t);
        den = fmaf(f, l[u], den);
#pragma unroll
        for (int i = 0; i < 4; i++) num[i] += f * x[u][i];
      }
    }
    if (redo || 32 * wave + n32 >= rows) continue;
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    uint16_t *op = a.out + head_row(a, it.row0, it.kv_head, row) * kD + 32 * db + 4 * h;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const Quad o = {(Value)(num[i][0] * inv), (Value)(num[i][1] * inv), (Value)(num[i][2] * inv), (Value)(num[i][3] * inv)};
      *reinterpret_cast<Quad *>(op + 8 * i) = o;
    }
  }
  redo_tiles<C, kD>(a, lds, flagged);
}

// Small tiles where every sequence's new tokens fit one: a second one reads K and V again,
// a large one has idle waves. (Small and large, us a call, 16 sequences of up to 4,096
// positions, 8 KV heads of 1, 2, 4 or 8 query heads: 16 rows a KV head 52 - 57 and
// 54 - 59, 32 rows 76 - 87 and 57 - 59, 64 rows 124 - 154 and 61 - 63. 2 KV heads of 16: 16
// rows 27 and 34, 32 rows 34 and 34, 64 rows 46 and 36. 48 sequences of one token of 2 heads
// 110 and 135. Of more than 16 query heads a KV head one token is more than a small tile:
// 17 to 32 heads 34, 128 heads 39.)
Variant variant_of(int group, int max_new) {
  return group <= kSmall.rows && (long long)group * max_new <= kSmall.rows ? kSmall : kLarge;
}

size_t workspace_of(const sh_paged_kv *kv, int heads, int max_new) {
  const Variant v = variant_of(heads / kv->kv_heads, max_new);
  return v.workers * (sizeof(MergeItem) + 2 * sizeof(int)) + (size_t)2 * v.workers * v.rows * (kv->head_dim + 2) * 4;
}

int check_attn_sizes(const sh_paged_kv *kv, int tokens, int heads, int max_new) {
  if (const char *wrong = check_paged_sizes(kv, tokens, heads)) return fail(SH_ERR_INVALID_ARGUMENT, "%s", wrong);
  if (!paged_dim_built(kv->head_dim))
    return fail(SH_ERR_UNSUPPORTED, "paged head_dim %d (64 or 128 are built)", kv->head_dim);
  if (max_new < 0) return fail(SH_ERR_INVALID_ARGUMENT, "max_new must not be negative");
  return SH_OK;
}

// A call of sh_attn_paged_* or of sh_attn_paged8_*, whose `kv` here is the sizes and
// index tensors of its cache, without pools.
struct AttnCall {
  const sh_paged_kv *kv;
  const uint16_t *q;
  uint16_t *out;
  int tokens, heads, max_new, window, sinks;
  float scale;
  void *workspace;
  size_t workspace_bytes;
};

int check_attn_call(sh_ctx *ctx, const AttnCall &c) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if ((rc = check_attn_sizes(c.kv, c.tokens, c.heads, c.max_new))) return rc;
  if (c.window < 0 || c.sinks < 0) return fail(SH_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
  // (times log2(e) it has to be finite)
  if (!(c.scale > 0.0f) || !(c.scale <= 0x1p127f))
    return fail(SH_ERR_INVALID_ARGUMENT, "scale must be positive and at most 2^127");
  return SH_OK;
}

// over_pools(p, bytes): whether that range lies over the cache.
template <class OverPools>
int check_attn_tensors(sh_ctx *ctx, const AttnCall &c, OverPools over_pools) {
  const size_t bytes = (size_t)c.tokens * c.heads * c.kv->head_dim * 2, need = workspace_of(c.kv, c.heads, c.max_new);
  int rc;
  if ((rc = check_range(ctx, c.q, bytes, "q")) || (rc = check_range(ctx, c.out, bytes, "out"))) return rc;
  if ((reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.out)) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
  if (ranges_overlap(c.q, bytes, c.out, bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "out overlaps q");
  if (c.workspace_bytes < need)
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer has %zu bytes, %zu are needed", c.workspace_bytes, need);
  if ((rc = check_range(ctx, c.workspace, need, "workspace"))) return rc;
  if (reinterpret_cast<uintptr_t>(c.workspace) & 15)
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer must be 16-byte aligned");
  if (ranges_overlap(c.workspace, need, c.q, bytes) || ranges_overlap(c.workspace, need, c.out, bytes) ||
      over_pools(c.workspace, need) || overlaps_index(c.kv, c.workspace, need))
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer overlaps a tensor of the call");
  if (overlaps_index(c.kv, c.out, bytes))
    return fail(SH_ERR_INVALID_ARGUMENT, "out overlaps the page table, lengths or starts");
  if (over_pools(c.out, bytes)) return fail(SH_ERR_INVALID_ARGUMENT, "out overlaps the cache");
  return SH_OK;
}

// All but the pools. small_unit: positions of a small tile's unit.
void fill_attn_args(const AttnCall &c, int small_unit, PagedAttnArgs *out) {
  PagedAttnArgs &a = *out;
  const sh_paged_kv *kv = c.kv;
  a.q = c.q;
  a.out = c.out;
  a.table = kv->page_table;
  a.heads = c.heads;
  a.group = c.heads / kv->kv_heads;
  a.group_inv = (65536 + a.group - 1) / a.group;
  a.max_pages = kv->max_pages;
  a.num_pages = kv->num_pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  const Variant v = variant_of(a.group, c.max_new);
  a.tile_rows = v.rows;
  a.scale_log2 = c.scale * 1.44269504f;
  a.no_score = a.scale_log2 <= kPlainScale ? -INFINITY : NAN;
  PagedPlan &p = a.plan;
  p.starts = kv->starts;
  p.lengths = kv->lengths;
  p.batch = kv->batch;
  p.tokens = c.tokens;
  p.kv_heads = kv->kv_heads;
  p.capacity = kv->max_pages * kv->page_size;
  p.per_tile = a.tile_rows / a.group;
  p.unit = v.rows == kSmall.rows ? small_unit : kLargeUnit;
  p.unit_shift = __builtin_ctz((unsigned)p.unit);
  p.window = c.window;
  p.sinks = c.sinks;
  p.min_piece = v.min_piece;
  p.workers = plan_workers(p.batch, p.kv_heads, c.tokens, p.capacity, p.per_tile, p.min_piece, v.workers);
  p.inv_workers = 1.0 / p.workers;
  p.whole_below = v.whole_below;
  a.items = static_cast<MergeItem *>(c.workspace);
  a.groups = reinterpret_cast<int *>(a.items + p.workers);
  a.redo = a.groups + p.workers;
  a.slots = reinterpret_cast<float *>(a.redo + p.workers);
}

}  // namespace
}  // namespace sh
