// Attention of new tokens over a KV cache in pages (sh_attn_paged_*): the kernels of
// 16-bit pages. What they share with others is in paged_attn.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "paged.h"
#include "paged_attn.h"
#include "paged_device.h"

namespace sh {
namespace {

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

// ---- the entry points ---------------------------------------------------------------

template <class T, int kD>
void launch(hipStream_t st, const PagedAttnArgs &a) {
  const int workers = a.plan.workers;
  if (a.tile_rows == kSmall.rows) {
    paged_small_kernel<T, kD><<<workers, kT, 0, st>>>(a);
    paged_merge_small_kernel<Pages16<T>, kD><<<workers, kMergeT, 0, st>>>(a);
    return;
  }
  paged_large_kernel<T, kD><<<workers, kT, 0, st>>>(a);
  paged_merge_large_kernel<Pages16<T>, kD><<<std::max(workers, 1024), kT, 0, st>>>(a);
}

template <class T>
int attn_paged(sh_ctx *ctx, const sh_paged_kv *kv, const uint16_t *q, uint16_t *out, int tokens, int heads,
               int max_new, int window, int sinks, float scale, void *workspace, size_t workspace_bytes) {
  const AttnCall c = {kv, q, out, tokens, heads, max_new, window, sinks, scale, workspace, workspace_bytes};
  int rc = check_attn_call(ctx, c);
  if (rc != SH_OK || tokens == 0 || kv->batch == 0) return rc;
  if ((rc = check_paged_pointers(ctx, kv)) || (rc = check_attn_tensors(ctx, c, [&](const void *p, size_t bytes) {
              const size_t pool = paged_pool_bytes(kv);
              return ranges_overlap(p, bytes, kv->k, pool) || ranges_overlap(p, bytes, kv->v, pool);
            })))
    return rc;
  PagedAttnArgs a;
  fill_attn_args(c, 32 * 128 / kv->head_dim, &a);
  a.k = kv->k;
  a.v = kv->v;
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
