// Attention of new tokens over a KV cache in pages of 8-bit values (sh_attn_paged8_*): the
// kernels that read such pages. How a call of many positions is divided, the merge and the
// tiles that matrix products cannot do are those of 16-bit pages (paged_attn.h).
//
// A byte times its row's power of two is a value of the 16-bit type but for that type's
// range, so the products, the softmax and their roundings are the same; only half the
// bytes are read.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "paged.h"
#include "paged_attn.h"
#include "paged_device.h"

namespace sh {
namespace {

struct Attn8Args : PagedAttnArgs {
  const uint8_t *pages;
  size_t page_bytes, v_at, v_scale_at;  // of a page: its bytes, the first row of V, the scales of V after those of K
};

// Pages of 8-bit values as attn_exact reads them.
template <class T>
struct Pages8 {
  typedef T Type;
  typedef Attn8Args Args;
  struct Row {
    long long at;  // of the row of K
    float k_scale, v_scale;
  };
  template <int kD>
  static __device__ __forceinline__ Row row(const Args &a, int page, int kv_head, int in_page) {
    const size_t first = (size_t)page * a.page_bytes, r = ((size_t)kv_head << a.page_shift) + in_page;
    const uint8_t *scale = a.pages + first + 2 * a.v_at + r;
    return Row{(long long)(first + r * kD), e8m0_scale(scale[0]), e8m0_scale(scale[a.v_scale_at])};
  }
  static __device__ __forceinline__ Row row_of_lane(Row r, int lane) {
    return Row{__shfl(r.at, lane, 64), __shfl(r.k_scale, lane, 64), __shfl(r.v_scale, lane, 64)};
  }
  static __device__ __forceinline__ float value(uint32_t byte, float scale) {
    return (float)__builtin_bit_cast(typename T::Pair, from_e4m3<T>(byte, scale).x)[0];
  }
  static __device__ __forceinline__ float k(const Args &a, Row r, int c) { return value(a.pages[r.at + c], r.k_scale); }
  static __device__ __forceinline__ float v(const Args &a, Row r, int c) {
    return value(a.pages[r.at + (long long)a.v_at + c], r.v_scale);
  }
};

// ---- tiles of up to 16 rows ------------------------------------------------------------
//
// As the kernel of 16-bit pages (paged_attn.hip), bound by the bytes of K and V: each
// wave takes units of 64 positions (128 at head_dim 64) by itself, twice as many as there
// for the same bytes in flight. What differs is how the values come to the products:
//  - K fragments straight from memory, 16 bytes of position lane % 16 per lane, which are
//    those of two products (of the 64 dims that four lanes hold, each product takes the
//    8 of each lane's half: q is read in the same order);
//  - V as 16-bit values to LDS rows, where a lane's 16 bytes have one scale.
// Both are converted with their scale in one instruction for two values. 48 tokens over up to
// 8,704 positions of 8 KV heads of 128 (640 MB) take 107 us, 6.0 TB/s, and a merge of 6; one
// over 777 12 us on 8 CUs.
template <int kD>
constexpr int kSmallUnit8 = 64 * 128 / kD;

template <class T, int kD>
struct SmallLds8 {
  union {
    uint8_t v[4][kSmallUnit8<kD> * kD * 2];
    float acc[4][kSmall.rows][kD];
  };
  float stat[4][kSmall.rows][2];
};

template <class T, int kD>
__device__ __forceinline__ bool attn_small8(const Attn8Args &a, const PagedTile &t, const TileSpan &s, int u0,
                                           int u1, int slot, SmallLds8<T, kD> &lds) {
  typedef typename T::Vec Vec;
  typedef typename T::Value Value;
  constexpr int kUnit = kSmallUnit8<kD>, kBlocks = kUnit / 16, kKL = kD / 64, kDT = kD / 16;
  constexpr int kRow = kD * 2, kChunks = kD / 16, kVLoads = kUnit * kChunks / 64, kVRows = 64 / kChunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, grp = lane >> 4, rows = s.count * a.group;
  const int row = min(r16, rows - 1), my_pos = s.pos0 + token_of(a, row);
  const uint16_t *qp = a.q + head_row(a, t.seq.row0 + s.first, t.kv_head, row) * kD + grp * 16;
  const int *table = a.table + (size_t)t.b * a.max_pages;
  const int last_pos = s.pos0 + s.count - 1, page_mask = (1 << a.page_shift) - 1;
  Vec q[2 * kKL];
#pragma unroll
  for (int kk = 0; kk < 2 * kKL; kk++) q[kk] = *reinterpret_cast<const Vec *>(qp + 64 * (kk / 2) + 8 * (kk % 2));

  // the table entry of block lane % kBlocks of unit j
  auto entry = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kUnit, min(j, u1 - 1)) + 16 * (lane % kBlocks);
    return table[min(p >> a.page_shift, a.max_pages - 1)];
  };
  u32x4 kr[kBlocks][kKL], vr[kVLoads];
  uint32_t ks[kBlocks], vs[kVLoads];  // the scales of the lane's rows
  size_t base[kBlocks], scales[kBlocks];  // of the blocks' first rows of K; bad: no page
  auto place = [&](int j, int entries, unsigned *bad) __attribute__((always_inline)) {
    const int p = span_position(s, kUnit, j);
    *bad = 0;
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++) {
      const int page = paged_page(__builtin_amdgcn_readlane(entries, tt), a.num_pages);
      if (page < 0) *bad |= 1u << tt;
      const size_t at = (size_t)max(page, 0) * a.page_bytes;
      const size_t row = ((size_t)t.kv_head << a.page_shift) + ((p + 16 * tt) & page_mask);
      base[tt] = at + row * kD;
      scales[tt] = at + 2 * a.v_at + row;
    }
  };
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int tt = 0; tt < kBlocks; tt++) {
#pragma unroll
      for (int c = 0; c < kKL; c++)
        kr[tt][c] = *reinterpret_cast<const u32x4 *>(a.pages + base[tt] + (r16 * kD + grp * 16 + 64 * c));
      ks[tt] = a.pages[scales[tt] + r16];
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kVLoads; u++) {
      const int block = u * kVRows / 16, r = u * kVRows % 16 + lane / kChunks;
      vr[u] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4 *>(a.pages + (base[block] + a.v_at) + (r * kD + (lane % kChunks) * 16)));
      vs[u] = a.pages[scales[block] + a.v_scale_at + r];
    }
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x4 acc[kDT];
#pragma unroll
  for (int dt = 0; dt < kDT; dt++) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint8_t *vl = lds.v[wave];
  // chunk c of row r lies at c ^ f(r): a transposing read's 32 lanes (8 rows, 2
  // chunks each) then hit 64 banks, and so do 16 lanes that write every other chunk
  auto swz = [](int r) { return kD == 128 ? 2 * (r & 7) + (r & 1) : 2 * ((r >> 1) & 3) + ((r >> 1) & 1); };
  const int ti = (lane >> 2) & 3, tq = lane & 3;
  int v_at[kDT];  // (f repeats every 8 rows)
  const int v_row = lane / kChunks, v_to = v_row * kRow + (((2 * (lane % kChunks)) ^ swz(v_row)) * 16);
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
    for (int c = 0; c < kKL; c++)
#pragma unroll
      for (int half = 0; half < 2; half++)
#pragma unroll
        for (int tt = 0; tt < kBlocks; tt++) {
          const u32x4 kf = from_e4m3<T>(kr[tt][c][2 * half], kr[tt][c][2 * half + 1], e8m0_scale(ks[tt]));
          sc[tt] = T::mfma16(__builtin_bit_cast(Vec, kf), q[2 * c + half], sc[tt]);
        }
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
        if (((bad >> (u * kVRows / 16)) & 1) || !tile_sees(a, s, p0 + u * kVRows + lane / kChunks)) {
          vr[u] = u32x4{0, 0, 0, 0};
          vs[u] = 0;
        }
    }
#pragma unroll
    for (int u = 0; u < kVLoads; u++) {
      const float scale = e8m0_scale(vs[u]);
      uint8_t *to = vl + u * kVRows * kRow;
      *reinterpret_cast<u32x4 *>(to + v_to) = from_e4m3<T>(vr[u].x, vr[u].y, scale);
      *reinterpret_cast<u32x4 *>(to + (v_to ^ 16)) = from_e4m3<T>(vr[u].z, vr[u].w, scale);
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
__global__ __launch_bounds__(kT, kSmall.workers / 256) void paged8_small_kernel(const Attn8Args a) {
  __shared__ __attribute__((aligned(16))) SmallLds8<T, kD> lds;
  __shared__ PlanLds plan;
  work_piece<false, 1, 1>(a, plan, [&](const PieceStep &st, Line) { return attn_small8<T, kD>(a, st.tile, st.span, st.u0, st.u1, st.slot, lds); });
}

// The sequence's tile without a place on the line (its units are all one workgroup's).
__device__ __forceinline__ PagedTile whole_tile(const Attn8Args &a, int b, int kv_head) {
  PagedTile t;
  t.seq = plan_seq(a.plan, b);
  for (int *v : {&t.seq.row0, &t.seq.n, &t.seq.len}) *v = uniform(*v);
  t.b = b;
  t.kv_head = kv_head;
  t.tile = 0;
  t.begin = t.cost = 0;
  return t;
}

// A call whose tiles are not cut: a workgroup a sequence and KV head (of as many new tokens
// as were announced one tile), nothing to plan and nothing to merge. What is not sound it
// does again.
template <class T, int kD>
__global__ __launch_bounds__(kT, kSmall.workers / 256) void paged8_small_whole_kernel(const Attn8Args a) {
  __shared__ __attribute__((aligned(16))) SmallLds8<T, kD> lds;
  for (int b = blockIdx.y; b < a.plan.batch; b += gridDim.y) {
    PagedTile t = whole_tile(a, b, blockIdx.x);
    const int tiles = plan_tiles(a.plan, t.seq);
    for (; t.tile < tiles; t.tile++) {
      const TileSpan s = plan_span(a.plan, t);
      if (!attn_small8<T, kD>(a, t, s, 0, s.units, -1, lds)) attn_exact<Pages8<T>, kD>(a, t, s);
    }
  }
}

// ---- tiles of up to 128 rows ------------------------------------------------------------
//
// As the kernel of 16-bit pages (paged_attn.hip): four waves of 32 rows share K and V units
// of 64 positions in LDS, double-buffered, a barrier per unit. Here a wave's 16 positions of
// a unit go through its registers: requested a unit ahead, converted to 16 bits among the
// next unit's products of scores (each value once, where fragments of bytes would be
// converted by all four waves) and written to the other buffer. Bound by the products and the
// softmax's vector work beside them: 8,192 tokens of 16 heads over 12,288 positions take 627 to
// 640 us at best, 860 to 880 TFLOP/s, and a merge of 16; a call 631 to 659 us, 834 to 871. (Units
// requested two ahead, or among other products: 629 to 638 where this took 627 to 631.)
constexpr float kSlack = 8.0f;

//
// kHalves 2: eight waves, four for the first half of the units and four for the others,
// whose sums are joined in LDS at the end.
template <int kD, int kHalves>
struct LargeLds8 {
  union {
    struct {
      uint8_t k[2 * kHalves][kLargeUnit * kD * 2], v[2 * kHalves][kLargeUnit * kD * 2];
    };
    f32x4 acc[4][kD / 8][64];  // of the other half: [wave][four sums][lane]
  };
  __attribute__((aligned(16))) unsigned bad[2 * kHalves][4];  // a 16-position block without a page
  float stat[4][2][64];
};

template <class T, int kD, int kHalves>
__device__ __forceinline__ bool attn_large8(const Attn8Args &a, const PagedTile &t, const TileSpan &s, int first,
                                           int end, int slot, LargeLds8<kD, kHalves> &lds) {
  typedef typename T::Vec Vec;
  typedef typename T::Value Value;
  typedef Value Quad __attribute__((ext_vector_type(4)));
  constexpr int kRow = kD * 2, kChunks = kD / 16, kKK = kD / 16, kDB = kD / 32;
  constexpr int kLoadRows = 64 / kChunks, kLoads = 16 / kLoadRows;  // of a wave's 16 positions
  const int lane = threadIdx.x & 63, half = kHalves == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
  const int middle = kHalves == 1 ? end : first + (end - first + 1) / 2;
  const int u0 = half == 0 ? first : middle, u1 = half == 0 ? middle : end;
  const auto buffer = [&](int j) { return 2 * half + (j & 1); };
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
  // hit all banks, 32 lanes of a transposing read of V (4 rows, 4 chunks each), and 16
  // that write every other chunk
  auto swz_k = [](int r) { return kD == 128 ? r & 15 : (r >> 1) & 7; };
  auto swz_v = [](int r) { return kD == 128 ? 4 * (r & 3) + (r & 1) : 4 * ((r >> 1) & 1) + ((r >> 1) & 1); };
  const int load_row = lane / kChunks, load_chunk = lane % kChunks;
  constexpr uint32_t kBuffer = kLargeUnit * kD * 2, kWave = 16 * kRow;
  // the table entry of this wave's 16 positions of unit j
  auto entry = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, min(j, u1 - 1)) + 16 * wave;
    return table[min(p >> a.page_shift, a.max_pages - 1)];
  };
  // this wave's 16 rows of K and V of unit j, requested; whether there is no page
  u32x4 kr[kLoads], vr[kLoads];
  uint32_t ks[kLoads], vs[kLoads];
  bool none = false;
  auto request = [&](int j, int e) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, j) + 16 * wave;
    const int page = paged_page(__builtin_amdgcn_readfirstlane(e), a.num_pages);
    none = page < 0;
    const size_t row = ((size_t)t.kv_head << a.page_shift) + (p & page_mask);
    const uint8_t *from = a.pages + (size_t)max(page, 0) * a.page_bytes;
    const uint8_t *rows = from + row * kD, *scales = from + 2 * a.v_at + row;
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
      kr[u] = *reinterpret_cast<const u32x4 *>(rows + (u * 1024 + lane * 16));
      vr[u] = *reinterpret_cast<const u32x4 *>(rows + a.v_at + (u * 1024 + lane * 16));
      ks[u] = scales[u * kLoadRows + load_row];
      vs[u] = scales[a.v_scale_at + u * kLoadRows + load_row];
    }
  };
  // load u of what was requested for unit j to its buffer; what no row sees is zeros
  // in V (of K, such scores are masked)
  auto keep_k = [&](int j, int u) __attribute__((always_inline)) {
    const int r = u * kLoadRows + load_row, at = wave * kWave + r * kRow + (((2 * load_chunk) ^ swz_k(r)) * 16);
    const float scale = e8m0_scale(ks[u]);
    *reinterpret_cast<u32x4 *>(lds.k[buffer(j)] + at) = from_e4m3<T>(kr[u].x, kr[u].y, scale);
    *reinterpret_cast<u32x4 *>(lds.k[buffer(j)] + (at ^ 16)) = from_e4m3<T>(kr[u].z, kr[u].w, scale);
  };
  auto keep_v = [&](int j, int u) __attribute__((always_inline)) {
    const int r = u * kLoadRows + load_row, at = wave * kWave + r * kRow + (((2 * load_chunk) ^ swz_v(r)) * 16);
    const float scale = e8m0_scale(vs[u]);
    *reinterpret_cast<u32x4 *>(lds.v[buffer(j)] + at) = from_e4m3<T>(vr[u].x, vr[u].y, scale);
    *reinterpret_cast<u32x4 *>(lds.v[buffer(j)] + (at ^ 16)) = from_e4m3<T>(vr[u].z, vr[u].w, scale);
  };
  auto blank = [&](int j) __attribute__((always_inline)) {
    const int p = span_position(s, kLargeUnit, j) + 16 * wave;
    if (lane == 0) lds.bad[buffer(j)][wave] = none ? 1 : 0;
    if (none || p + 16 > s.hi || (a.plan.window > 0 && p < s.lo && p + 16 > s.sinks)) {
#pragma unroll
      for (int u = 0; u < kLoads; u++) {
        if (none || !tile_sees(a, s, p + u * kLoadRows + load_row)) {
          vr[u] = u32x4{0, 0, 0, 0};
          vs[u] = 0;
        }
      }
    }
  };
  auto keep = [&](int j) __attribute__((always_inline)) {
    blank(j);
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
      keep_k(j, u);
      keep_v(j, u);
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
    request(u0, entry(u0));
    entries = entry(u0 + 1);
    keep(u0);
    if (u0 + 1 < u1) request(u0 + 1, entries);
    entries = entry(u0 + 2);
  }
  const int ti = (lane >> 2) & 3, tq = lane & 3, side = (lane >> 4) & 1;
  const int v_at0 = (4 * h + ti) * kRow + (((2 * side + (tq >> 1)) ^ swz_v(4 * h + ti)) * 16) + (tq & 1) * 8;
  const int k_at0 = n32 * kRow + ((h ^ swz_k(n32)) * 16);
  if (!active) {  // a wave without rows loads its part
    for (int j = u0; j < u1; j++) {
      lds_barrier();
      if (j + 1 < u1) keep(j + 1);
      if (j + 2 < u1) request(j + 2, entries);
      entries = entry(j + 3);
    }
  }
  for (int j = active ? u0 : u1; j < u1; j++) {
    const int p0 = span_position(s, kLargeUnit, j), buf = buffer(j), next = min(j + 1, u1 - 1);
    lds_barrier();
    if (j + 1 < u1) blank(next);
    // Fragments are requested ahead of the products that take them (the compiler left
    // to itself reads each just before its use), and the next unit's values converted
    // and written among the products of the scores. (Of the last unit, what there is once
    // more, to the buffer that nobody reads.)
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
      if (kk % 4 == 1) keep_k(j + 1, kk / 4);
      if (kk % 4 == 3) keep_v(j + 1, kk / 4);
      __builtin_amdgcn_sched_barrier(0);
    }
    static_assert(kLoads == kKK / 4, "a load of K or V every other step");
    if (j + 2 < u1) request(j + 2, entries);
    entries = entry(j + 3);
    // (a wave in its softmax before one in its products, which take turns)
    __builtin_amdgcn_s_setprio(1);
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
  if constexpr (kHalves == 2) {
    if (u1 - u0 < middle - first) lds_barrier();  // (the others had a unit more)
    lds_barrier();  // K and V are read
    if (half == 1 && active) {
#pragma unroll
      for (int db = 0; db < kDB; db++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          lds.acc[wave][4 * db + i][lane] = f32x4{acc[db][4 * i], acc[db][4 * i + 1], acc[db][4 * i + 2], acc[db][4 * i + 3]};
      lds.stat[wave][0][lane] = m_run;
      lds.stat[wave][1][lane] = l_run;
    }
    lds_barrier();
    if (half == 0 && active) {
      const float other_m = lds.stat[wave][0][lane], other_l = lds.stat[wave][1][lane], m = fmaxf(m_run, other_m);
      const float mine = m_run == m ? 1.0f : exp2_weight(m_run - m), other = other_m == m ? 1.0f : exp2_weight(other_m - m);
      m_run = m;
      l_run = fmaf(other_l, other, l_run * mine);
#pragma unroll
      for (int db = 0; db < kDB; db++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 x = lds.acc[wave][4 * db + i][lane];
#pragma unroll
          for (int e = 0; e < 4; e++) acc[db][4 * i + e] = fmaf(x[e], other, acc[db][4 * i + e] * mine);
        }
    }
  }
  bool sound = true;
  const bool there = half == 0 && 32 * wave + n32 < rows;
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
__global__ __launch_bounds__(kT, kLarge.workers / 256) void paged8_large_kernel(const Attn8Args a) {
  __shared__ __attribute__((aligned(16))) LargeLds8<kD, 1> lds;
  __shared__ PlanLds plan;
  work_piece<true, 32, kD / 32>(a, plan, [&](const PieceStep &st, Line) {
    return attn_large8<T, kD, 1>(a, st.tile, st.span, st.u0, st.u1, st.slot, lds);
  });
}

// find_tile's wave. Sums by lane moves as in wave_scan_line.
struct DeviceWave {
  typedef int Int;
  template <class F>
  static __device__ __forceinline__ Int each(F f) {
    return f((int)(threadIdx.x & 63));
  }
  template <class F>
  static __device__ __forceinline__ Int map(Int v, F f) {
    return f(v);
  }
  static __device__ __forceinline__ Int scan(Int v) {
    const auto add = [&](int moved) { v = min(v + moved, kMaxTiles); };
    add(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
    return v;
  }
  static __device__ __forceinline__ int read(Int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
  template <class F>
  static __device__ __forceinline__ uint64_t ballot(Int v, F f) {
    return __ballot(f(v));
  }
  static __device__ __forceinline__ int nth(uint64_t those, int n) {
    const int rank = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(those >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)those, 0));
    return __builtin_ctzll(__ballot((those >> (threadIdx.x & 63) & 1) != 0 && rank == n));
  }
};

// A call whose tiles are not cut: a workgroup a tile. (With places between the sequences that
// have no tile, so that no sums were needed, 16 sequences of 256 new tokens took 67 us and not
// 49: which CU a workgroup goes to is settled by its number, and some had two rounds.)
template <class T, int kD, int kHalves>
__global__ __launch_bounds__(kHalves * kT, 2) void paged8_large_whole_kernel(const Attn8Args a) {
  __shared__ __attribute__((aligned(16))) LargeLds8<kD, kHalves> lds;
  for (int tile = blockIdx.y, total = tile + 1; tile < total; tile += gridDim.y) {
    int back = 0;
    const int b = uniform(find_tile<DeviceWave>(a.plan, tile, &back, &total));
    if (b < 0) return;
    PagedTile t = whole_tile(a, b, blockIdx.x);
    t.tile = plan_tiles(a.plan, t.seq) - 1 - uniform(back);
    const TileSpan s = plan_span(a.plan, t);
    if (!attn_large8<T, kD, kHalves>(a, t, s, 0, s.units, -1, lds)) attn_exact<Pages8<T>, kD>(a, t, s);
  }
}

// ---- the entry points ---------------------------------------------------------------

// Where tiles see few positions they are not cut: to plan the pieces takes 4 us, and the
// merge, a launch that reads all parts, 4 to 50. Up to 18 units (tables of 1,024 positions
// and some pages more, of 16-row tiles at head_dim 64 of 2,048) always, up to 34 where there
// are tiles for every CU, so that a long one matters less. Cut and not, us a call:
// - a token each, 16-row tiles: 1 sequence of 8 KV heads of 128 over 128 positions 13.1 and
//   5.6, 512 13.3 and 8.5, 1,024 13.7 and 12.5, 2,048 13.7 and 19.1; 48 of them over up to
//   256 22.1 and 10.5, 1,024 30.6 and 23.0, 2,048 42.1 and 37.4, 4,096 69.6 and 68.9; 64 of
//   12 KV heads of 64 over up to 512 29.5 and 19.9, 2,048 47.5 and 41.2; a window of 256 of
//   up to 4,096, 16 of 8 KV heads of 128 20.0 and 11.0;
// - chunks, 128-row tiles: 8 prompts of 512 of 12 KV heads of 64 36.7 and 20.5, 1 of 1,024 23.6
//   and 25.8; of 8 KV heads of 128, 512 new tokens after 512 29.8 and 32.8, after 1,536 40 and
//   56, 16 times 256 after up to 768 88 and 51, 4 prompts of 2,048 149 and 106, 4 of 4,096 408
//   and 322, but 40 times 64 after up to 4,032 122 and 145; 63 single tokens and a prompt of
//   1,024 83 and 58.
// Two halves of a workgroup share a 128-row tile's units where there can be no more tiles than
// CUs and there are units enough for the join. One and two halves: 1 prompt of 1,024 of 12 KV
// heads of 64 25.9 and 21.3, 4 of up to 633 19.9 and 17.9, 8 of 1,024 41.5 and 50.0; of 8 KV
// heads of 128, 512 new tokens after 512 32.7 and 28.3, 1 prompt of 256 14.6 and 15.0, of 512
// 20.7 and 19.6. (8 ragged prompts of up to 333 over 1,024, some 250 tiles of 64: 29 and 36.)
// (Eight waves for a 16-row tile: as long, a CU reads no faster. Tiles not cut but on planned
// pieces: 1 sequence over 128 7.1, 16 14.4, 8 prompts of 512 38.)
template <class T, int kD>
void launch8(hipStream_t st, const Attn8Args &a) {
  const PagedPlan &p = a.plan;
  const bool small = a.tile_rows == kSmall.rows;
  const long long seen = p.window > 0 ? std::min((long long)p.sinks + p.window, (long long)p.capacity) : p.capacity;
  const long long tiles = (long long)std::max(p.batch, p.tokens / p.per_tile) * p.kv_heads;
  if ((small || p.batch <= kMaxWholeBatch) && seen <= (tiles >= 256 ? 34 : 18) * p.unit) {
    if (small) {
      paged8_small_whole_kernel<T, kD><<<dim3(p.kv_heads, std::min(p.batch, 32768)), kT, 0, st>>>(a);
    } else {
      const int most = p.batch + p.tokens / p.per_tile;  // tiles (of starts in order; any others are found too)
      const dim3 grid(p.kv_heads, std::min(most, 32768));
      if ((long long)most * p.kv_heads <= 256 && seen > 4 * p.unit)
        paged8_large_whole_kernel<T, kD, 2><<<grid, 2 * kT, 0, st>>>(a);
      else
        paged8_large_whole_kernel<T, kD, 1><<<grid, kT, 0, st>>>(a);
    }
    return;
  }
  if (small) {
    paged8_small_kernel<T, kD><<<p.workers, kT, 0, st>>>(a);
    paged_merge_small_kernel<Pages8<T>, kD><<<p.workers, kMergeT, 0, st>>>(a);
  } else {
    paged8_large_kernel<T, kD><<<p.workers, kT, 0, st>>>(a);
    paged_merge_large_kernel<Pages8<T>, kD><<<std::max(p.workers, 1024), kT, 0, st>>>(a);
  }
}

template <class T>
int attn_paged8(sh_ctx *ctx, const sh_paged_kv8 *kv, const uint16_t *q, uint16_t *out, int tokens, int heads,
                int max_new, int window, int sinks, float scale, void *workspace, size_t workspace_bytes) {
  if (!kv) return fail(SH_ERR_INVALID_ARGUMENT, "the paged cache is NULL");
  const sh_paged_kv index = paged8_index(kv);
  const AttnCall c = {&index, q, out, tokens, heads, max_new, window, sinks, scale, workspace, workspace_bytes};
  int rc = check_attn_call(ctx, c);
  if (rc != SH_OK || tokens == 0 || kv->batch == 0) return rc;
  if ((rc = check_paged8_pointers(ctx, kv)) || (rc = check_attn_tensors(ctx, c, [&](const void *p, size_t bytes) {
              return ranges_overlap(p, bytes, kv->pages, paged8_pool_bytes(kv));
            })))
    return rc;
  Attn8Args a;
  fill_attn_args(c, 64 * 128 / kv->head_dim, &a);
  a.k = a.v = nullptr;
  a.pages = kv->pages;
  a.page_bytes = paged8_page_bytes(kv);
  a.v_scale_at = (size_t)kv->kv_heads * kv->page_size;
  a.v_at = a.v_scale_at * kv->head_dim;
  const hipStream_t st = stream_of(ctx);
  if (kv->head_dim == 64)
    launch8<T, 64>(st, a);
  else
    launch8<T, 128>(st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SH_OK : hip_fail(e, "attn_paged8");
}

}  // namespace
}  // namespace sh

using namespace sh;

extern "C" {

SH_API int sh_attn_paged8_workspace(const sh_paged_kv8 *kv, int tokens, int heads, int max_new, size_t *bytes) {
  if (!bytes) return fail(SH_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (!kv) return fail(SH_ERR_INVALID_ARGUMENT, "the paged cache is NULL");
  const sh_paged_kv index = paged8_index(kv);
  const int rc = check_attn_sizes(&index, tokens, heads, max_new);
  if (rc != SH_OK) return rc;
  *bytes = workspace_of(&index, heads, max_new);
  return SH_OK;
}

SH_API int sh_attn_paged8_f16(sh_ctx *ctx, const sh_paged_kv8 *kv, const uint16_t *q, uint16_t *out, int tokens,
                              int heads, int max_new, int window, int sinks, float scale, void *workspace,
                              size_t workspace_bytes) {
  return attn_paged8<PagedF16>(ctx, kv, q, out, tokens, heads, max_new, window, sinks, scale, workspace,
                               workspace_bytes);
}

SH_API int sh_attn_paged8_bf16(sh_ctx *ctx, const sh_paged_kv8 *kv, const uint16_t *q, uint16_t *out, int tokens,
                               int heads, int max_new, int window, int sinks, float scale, void *workspace,
                               size_t workspace_bytes) {
  return attn_paged8<PagedBf16>(ctx, kv, q, out, tokens, heads, max_new, window, sinks, scale, workspace,
                                workspace_bytes);
}

}  // extern "C"
