// Attention of new tokens over a KV cache in pages (sh_attn_paged_*).
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

// A tile in fp32, a wave per row, a lane per position of 64: whatever the values are.
// The maximum is q.k's, the scale taken after it is subtracted, so that the largest
// weight is 1 however large the scores; the V sums are those of weights divided by their
// sum so far, and so no larger than the values. A score of -infinity, and a weight that
// is 0 in fp32, adds nothing. For tiles that the matrix products cannot do, and slow:
// each lane reads a row of K of its own, and a worker with one such tile has all of its
// tiles done again. A NaN that one of 48 decode rows of up to 4,352 positions sees:
// 0.11 -> 4.0 ms; one in the last of 8,192 tokens over 12,288 positions: 0.6 -> 285 ms.
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
        bool seen = p < end && Sees(a, s, pos, p)(0);
        long long at = 0;  // of the position's k and v
        if (seen) {
          const int page = paged_page(a.table[(size_t)t.b * a.max_pages + (p >> a.page_shift)], a.num_pages);
          seen = page >= 0;
          at = (((((long long)max(page, 0) * a.plan.kv_heads + t.kv_head) << a.page_shift) +
                 (p & ((1 << a.page_shift) - 1))) * kD);
        }
        float dot = -INFINITY;
        if (seen) {
          dot = 0.0f;
          for (int c = 0; c < kD; c++) dot = fmaf((float)q[c], (float)kp[at + c], dot);
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
          const long long ai = __shfl(at, i, 64);
          if (wi == 0.0f) continue;
#pragma unroll
          for (int j = 0; j < kDims; j++) acc[j] = fmaf(wi, (float)vp[ai + lane + 64 * j], acc[j]);
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
// 48 ragged sequences of up to 4,352 positions (626 MB of bf16): 101 us here and 6 in
// the merge, 6.2 TB/s of a copy's 6.4. 16 of up to 16,000 positions 134 us a call, with a
// window of 1,024 and 4 sinks 25.
template <int kD>
constexpr int kSmallUnit = 32 * 128 / kD;

template <class T, int kD>
struct SmallLds {
  union {
    uint8_t v[4][kSmallUnit<kD> * kD * 2];
    float acc[4][kSmall.rows][kD];
  };
  float stat[4][kSmall.rows][2];
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
  // (V as what the caches need not keep: 48 ragged sequences of up to 4,352 positions
  // 122 -> 112 us a call, of that length all 154 -> 143. K as well: 110 and 152, and 48
  // sequences of the same pages 84 -> 90.)
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kVLoads; u++)
      vr[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(
          a.v + base[u * kVRows / 16] + ((u * kVRows % 16 + lane / kChunks) * kD + (lane % kChunks) * 8)));
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
      const Sees seen(a, s, my_pos, p0 + 4 * grp);
#pragma unroll
      for (int tt = 0; tt < kBlocks; tt++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (((bad >> tt) & 1) || !seen(16 * tt + e)) sc[tt][e] = -INFINITY;
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
        p[tt / 2][(tt & 1) * 4 + e] = (Value)exp2_weight(fmaf(sc[tt][e], a.scale_log2, -off));
      }
#pragma unroll
    for (int i = 0; i < kBlocks / 2; i++) ls = T::sum8(p[i], ls);
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
  bool sound = true;
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
    sound = sound && score_fits<T>(a, m) && sum_fits(sum) && l < INFINITY;
    store_value<T, kD>(a, t, s, slot, r, dim, sum, l);
    if (slot >= 0 && dim == 0) {
      slot_stats<kD>(a, slot, r)[0] = m;
      slot_stats<kD>(a, slot, r)[1] = l;
    }
  }
  return !__syncthreads_or(sound ? 0 : 1);
}

template <class T, int kD>
__global__ __launch_bounds__(kT, kSmall.workers / 256) void paged_small_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) SmallLds<T, kD> lds;
  __shared__ PlanLds plan;
  work_piece<false, 1, 1>(a, plan, [&](const PieceStep &st, Line) { return attn_small<T, kD>(a, st.tile, st.span, st.u0, st.u1, st.slot, lds); });
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
// 8,192 tokens over 12,288 positions, 16 heads of 128 (550 GFLOP): 590 to 620 us a call
// with the merge, 890 to 930 TFLOP/s, where a large product reaches 1,228; matrix cores
// busy 41 % of the time, vector units (the softmax) 40 %, mostly in turn.
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
  // (both f only flip bits of the chunk that a load, a step kk or a block db counts
  // up, so that one offset each serves all of them)
  const int load_row = lane / kChunks, load_chunk = lane % kChunks;
  const uint32_t k_off = load_row * kRow + ((load_chunk ^ swz_k(load_row)) * 16);
  const uint32_t v_off = load_row * kRow + ((load_chunk ^ swz_v(load_row)) * 16);
  const uint32_t k_lds = (uint32_t)(uintptr_t)(SH_PAGED_LDS uint8_t *)lds.k[0];
  const uint32_t v_lds = (uint32_t)(uintptr_t)(SH_PAGED_LDS uint8_t *)lds.v[0];
  constexpr uint32_t kBuffer = kLargeUnit * kD * 2, kWave = 16 * kRow;
  // the table entry of this wave's 16 positions of unit j
  auto entry = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, min(j, u1 - 1)) + 16 * wave;
    return table[min(p >> a.page_shift, a.max_pages - 1)];
  };
  // this wave's 16 rows of K and V of unit j (their addresses; whether there is no
  // page), then load u of them to buffer j & 1, or nothing. (Inline asm: through the
  // compiler's builtin, later LDS reads would wait for every load in flight. The branch
  // is inside, so that the products around it stay one block to the scheduler.)
  uint64_t k_from = 0, v_from = 0;
  uint32_t to = 0;
  auto place = [&](int j, int e) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, j) + 16 * wave;
    const int page = paged_page(__builtin_amdgcn_readfirstlane(e), a.num_pages);
    if (lane == 0) lds.bad[j & 1][wave] = page < 0 ? 1 : 0;
    const size_t at = ((((size_t)max(page, 0) * a.plan.kv_heads + t.kv_head) << a.page_shift) + (p & page_mask)) * kRow;
    k_from = (uint64_t)(uintptr_t)a.k + at;
    v_from = (uint64_t)(uintptr_t)a.v + at;
    to = (j & 1) * kBuffer + wave * kWave;
    return page < 0;
  };
  auto load = [&](int u, int really) __attribute__((always_inline)) {
    asm volatile(
        "s_cmp_eq_u32 %6, 0\n\t"
        "s_cbranch_scc1 .Lpaged_load%=\n\t"
        "s_mov_b32 m0, %4\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %2\n\t"
        "s_mov_b32 m0, %5\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %3\n"
        ".Lpaged_load%=:"
        ::"v"(k_off ^ (64 * u)), "v"(v_off), "s"(k_from + u * 1024), "s"(v_from + u * 1024),
        "s"(k_lds + to + u * 1024), "s"(v_lds + to + u * 1024), "s"(uniform(really))
        : "memory", "scc", "m0");
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16 acc[kDB];
#pragma unroll
  for (int db = 0; db < kDB; db++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[db][i] = 0.0f;

  __syncthreads();  // the last tile's LDS reads are done
  int entries = 0;
  bool none = false;  // this wave's 16 positions have no page
  if (u0 < u1) {
    none = place(u0, entry(u0));
#pragma unroll
    for (int u = 0; u < kLoads; u++) load(u, 1);
    entries = entry(u0 + 1);
  }
  const int ti = (lane >> 2) & 3, tq = lane & 3, side = (lane >> 4) & 1;
  const int v_at0 = (4 * h + ti) * kRow + (((2 * side + (tq >> 1)) ^ swz_v(4 * h + ti)) * 16) + (tq & 1) * 8;
  const int k_at0 = n32 * kRow + ((h ^ swz_k(n32)) * 16);
  // the loads of unit j are here and what no row sees is zeros in V
  auto arrive = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, j) + 16 * wave;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (none || p + 16 > s.hi || (a.plan.window > 0 && p < s.lo && p + 16 > s.sinks)) {
#pragma unroll
      for (int u = 0; u < kLoads; u++) {
        if (none || !tile_sees(a, s, p + u * kLoadRows + load_row))
          *reinterpret_cast<u32x4 *>(&lds.v[j & 1][wave * kWave + u * 1024 + lane * 16]) = u32x4{0, 0, 0, 0};
      }
    }
    lds_barrier();
  };
  if (!active) {  // a wave without rows loads its part
    for (int j = u0; j < u1; j++) {
      arrive(j);
      if (j + 1 < u1) {
        none = place(j + 1, entries);
#pragma unroll
        for (int u = 0; u < kLoads; u++) load(u, 1);
        entries = entry(j + 2);
      }
    }
  }
  for (int j = active ? u0 : u1; j < u1; j++) {
    const int p0 = span_position(s, kLargeUnit, j), buf = j & 1, more = j + 1 < u1 ? 1 : 0;
    arrive(j);
    // Fragments are requested ahead of the products that take them (the compiler left
    // to itself reads each just before its use), and the next unit's loads spread over
    // the products of the scores (requested together they held the wave up for a fifth
    // of the unit).
    Vec kf[2][kKK];
    s16x4 vh[4][kDB][2];
    const int k_at = k_at0 + buf * (int)kBuffer, v_at = v_at0 + buf * (int)kBuffer;
    auto read_v = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < kDB; db++)
#pragma unroll
        for (int q2 = 0; q2 < 2; q2++)
          vh[ks][db][q2] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (SH_PAGED_LDS s16x4 *)((SH_PAGED_LDS uint8_t *)lds.v[0] + (v_at ^ (64 * db)) + (16 * ks + 8 * q2) * kRow));
    };
    auto read_k = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
      for (int sb = 0; sb < 2; sb++)
        kf[sb][kk] = *reinterpret_cast<const Vec *>(lds.k[0] + (k_at ^ (32 * kk)) + 32 * sb * kRow);
    };
    constexpr int kAhead = 4;
#pragma unroll
    for (int kk = 0; kk < kAhead; kk++) read_k(kk);
    const u32x4 bad4 = *reinterpret_cast<const u32x4 *>(lds.bad[buf]);
    __builtin_amdgcn_sched_barrier(0);
    f32x16 sc[2];
#pragma unroll
    for (int sb = 0; sb < 2; sb++)
#pragma unroll
      for (int i = 0; i < 16; i++) sc[sb][i] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < kKK; kk++) {
#pragma unroll
      for (int sb = 0; sb < 2; sb++) sc[sb] = T::mfma32(kf[sb][kk], q[kk], sc[sb]);
      __builtin_amdgcn_sched_barrier(0);
      if (kk + kAhead < kKK) read_k(kk + kAhead);
      if (kk == 0) none = place(min(j + 1, u1 - 1), entries);
      if (kk % 2 == 1) load(kk / 2, more);
      __builtin_amdgcn_sched_barrier(0);
    }
    static_assert(kLoads == kKK / 2, "a pair of loads every other step");
    // (a wave in its softmax before one in its products, which take turns: 610 -> 599 us
    // for 8,192 tokens over 12,288 positions)
    __builtin_amdgcn_s_setprio(1);
    entries = entry(j + 2);
    read_v(0);
    read_v(1);
    __builtin_amdgcn_sched_barrier(0);
    const unsigned bad = __builtin_amdgcn_readfirstlane(bad4.x | (bad4.y << 1) | (bad4.z << 2) | (bad4.w << 3));
    const bool plain = bad == 0 && p0 + kLargeUnit <= pos_lo + 1 &&
                       (a.plan.window == 0 || p0 > pos_hi - a.plan.window || p0 + kLargeUnit <= s.sinks);
    if (!plain) {
      const Sees seen(a, s, my_pos, p0 + 4 * h);
#pragma unroll
      for (int sb = 0; sb < 2; sb++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (((bad >> (2 * sb + i / 8)) & 1) || !seen(32 * sb + 8 * (i / 4) + i % 4)) sc[sb][i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < 2; sb++)
#pragma unroll
      for (int i = 0; i < 16; i++) mx = fmaxf(mx, sc[sb][i]);
    mx = half_max(mx) * a.scale_log2;
    // the sums are rescaled only once a row's maximum has grown by 2^kSlack: until then
    // its weights are up to 2^kSlack times as large
    const int grown = uniform(__any(mx > m_run + kSlack) ? 1 : 0);
    const float m = grown ? fmaxf(m_run, mx) : m_run;
    const float corr = m_run == m ? 1.0f : exp2_weight(m_run - m);
    m_run = m;
    l_run *= corr;
    scale_if(acc, corr, grown);
    // (a row that has seen nothing yet: its weights are exp2(-infinity))
    const float off = (m_run == -INFINITY ? 0.0f : m_run) - T::kWeightLog2;
    float ls = 0.0f;
    Vec p[4];
#pragma unroll
    for (int sb = 0; sb < 2; sb++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        p[2 * sb + i / 8][i % 8] = (Value)exp2_weight(fmaf(sc[sb][i], a.scale_log2, -off));
      }
    ls = T::sum8(p[1], T::sum8(p[0], ls));
    l_run += ls + T::sum8(p[3], T::sum8(p[2], 0.0f));
    __builtin_amdgcn_sched_barrier(0);
    read_v(2);
    read_v(3);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
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
  bool sound = true;
  const bool there = 32 * wave + n32 < rows;
  if (there) sound = score_fits<T>(a, m_run) && l_run < INFINITY;
  const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
  uint16_t *op = a.out + head_row(a, t.seq.row0 + s.first, t.kv_head, row) * kD;
#pragma unroll
  for (int db = 0; db < kDB; db++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x4 x = {acc[db][4 * i], acc[db][4 * i + 1], acc[db][4 * i + 2], acc[db][4 * i + 3]};
#pragma unroll
      for (int e = 0; e < 4; e++) sound = sound && (!there || sum_fits(x[e]));
      if (slot >= 0) {
        if (active) *slot_large<kD>(a, slot, wave, db, i) = x;
      } else if (there) {
        const Quad o = {(Value)(x[0] * inv), (Value)(x[1] * inv), (Value)(x[2] * inv), (Value)(x[3] * inv)};
        *reinterpret_cast<Quad *>(op + 32 * db + 8 * i + 4 * h) = o;
      }
    }
  if (slot >= 0 && there && h == 0) {
    slot_stats<kD>(a, slot, row)[0] = m_run;
    slot_stats<kD>(a, slot, row)[1] = l_run;
  }
  return !__syncthreads_or(sound ? 0 : 1);
}

template <class T, int kD>
__global__ __launch_bounds__(kT, kLarge.workers / 256) void paged_large_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) LargeLds<kD> lds;
  __shared__ PlanLds plan;
  work_piece<true, 32, kD / 32>(a, plan, [&](const PieceStep &st, Line) {
    return attn_large<T, kD>(a, st.tile, st.span, st.u0, st.u1, st.slot, lds);
  });
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
template <class T, int kD>
__device__ __forceinline__ void redo_tiles(const PagedAttnArgs &a, MergeLds &lds, int flagged) {
  int w = blockIdx.x;
  if (flagged == 0) return;
  __syncthreads();  // lds.prefix is read
  MergeItem unused;
  walk_piece<false>(a.plan, &w, lds.plan, &unused, [&](const PieceStep &st, Line piece) {
    if (st.slot >= 0)  // a cut tile is the first flagged worker's
      for (int j = plan_first(st.tile, w, piece, w * piece); j < w; j++)
        if (a.redo[j] != 0) return true;
    attn_exact<T, kD>(a, st.tile, st.span);
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
template <class T, int kD>
__global__ __launch_bounds__(kMergeT) void paged_merge_small_kernel(const PagedAttnArgs a) {
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
  redo_tiles<T, kD>(a, lds, flagged);
}

template <class T, int kD>
__global__ __launch_bounds__(kT) void paged_merge_large_kernel(const PagedAttnArgs a) {
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
  redo_tiles<T, kD>(a, lds, flagged);
}

// ---- the entry points ---------------------------------------------------------------

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

template <class T, int kD>
void launch(hipStream_t st, const PagedAttnArgs &a) {
  const int workers = a.plan.workers;
  if (a.tile_rows == kSmall.rows) {
    paged_small_kernel<T, kD><<<workers, kT, 0, st>>>(a);
    paged_merge_small_kernel<T, kD><<<workers, kMergeT, 0, st>>>(a);
    return;
  }
  paged_large_kernel<T, kD><<<workers, kT, 0, st>>>(a);
  paged_merge_large_kernel<T, kD><<<std::max(workers, 1024), kT, 0, st>>>(a);
}

template <class T>
int attn_paged(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *q, uint16_t *out, int tokens, int heads,
               int max_new, int window, int sinks, float scale, void *workspace, size_t workspace_bytes) {
  int rc = enter(ctx);
  if (rc != SH_OK) return rc;
  if ((rc = check_attn_sizes(kv, tokens, heads, max_new))) return rc;
  if (window < 0 || sinks < 0) return fail(SH_ERR_INVALID_ARGUMENT, "window and sinks must not be negative");
  // (times log2(e) it has to be finite)
  if (!(scale > 0.0f) || !(scale <= 0x1p127f))
    return fail(SH_ERR_INVALID_ARGUMENT, "scale must be positive and at most 2^127");
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
  const size_t pool = paged_pool_bytes(kv);
  if (ranges_overlap(workspace, need, q, bytes) || ranges_overlap(workspace, need, out, bytes) ||
      ranges_overlap(workspace, need, kv->k, pool) || ranges_overlap(workspace, need, kv->v, pool) ||
      overlaps_index(kv, workspace, need))
    return fail(SH_ERR_INVALID_ARGUMENT, "the work buffer overlaps a tensor of the call");
  if (overlaps_index(kv, out, bytes))
    return fail(SH_ERR_INVALID_ARGUMENT, "out overlaps the page table, lengths or starts");
  if (ranges_overlap(out, bytes, kv->k, pool) || ranges_overlap(out, bytes, kv->v, pool))
    return fail(SH_ERR_INVALID_ARGUMENT, "out overlaps the cache");
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
  const Variant v = variant_of(a.group, max_new);
  a.tile_rows = v.rows;
  a.scale_log2 = scale * 1.44269504f;
  a.no_score = a.scale_log2 <= kPlainScale ? -INFINITY : NAN;
  PagedPlan &p = a.plan;
  p.starts = kv->starts;
  p.lengths = kv->lengths;
  p.batch = kv->batch;
  p.tokens = tokens;
  p.kv_heads = kv->kv_heads;
  p.capacity = kv->max_pages * kv->page_size;
  p.per_tile = a.tile_rows / a.group;
  p.unit = v.rows == kSmall.rows ? 32 * 128 / kv->head_dim : kLargeUnit;
  p.unit_shift = __builtin_ctz((unsigned)p.unit);
  p.window = window;
  p.sinks = sinks;
  p.min_piece = v.min_piece;
  p.workers = plan_workers(p.batch, p.kv_heads, tokens, p.capacity, p.per_tile, p.min_piece, v.workers);
  p.inv_workers = 1.0 / p.workers;
  a.items = static_cast<MergeItem *>(workspace);
  a.groups = reinterpret_cast<int *>(a.items + p.workers);
  a.redo = a.groups + p.workers;
  a.slots = reinterpret_cast<float *>(a.redo + p.workers);
  p.whole_below = v.whole_below;
  const hipStream_t st = stream_of(ctx);
  if (kv->head_dim == 64)
    launch<T, 64>(st, a);
  else
    launch<T, 128>(st, a);
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
