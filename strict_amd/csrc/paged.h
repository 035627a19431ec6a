// A KV cache in pages: which rows and positions a batch's sequences have, how
// the attention over them is divided among workgroups, and the argument checks
// of the paged operators that need no device. Plain C++ on host and device, so
// that the bounds below are checked on the CPU for any device data (tests/cpp).
//
// What lies in device memory (starts, lengths, page table) cannot be checked on
// the host: every value is brought into its range here before it indexes
// anything, and a page number out of range makes its positions invisible.
#pragma once

#include <cstddef>
#include <cstdint>

#include "strict_hip.h"

#if defined(__HIPCC__)
#define SH_HD __host__ __device__ __forceinline__
#else
#define SH_HD inline
#endif

namespace sh {

constexpr int kMaxPagedTokens = 1 << 22, kMaxPagedBatch = 1 << 16, kMaxPagedKvHeads = 1 << 10;
constexpr int kMaxPagedPositions = 1 << 28;  // max_pages * page_size

// a / b for 0 <= a, 0 < b; most are small, and a 64-bit division is some hundred
// instructions.
SH_HD long long plan_div(long long a, long long b) {
  if (((a | b) >> 31) == 0) return (long long)((uint32_t)a / (uint32_t)b);
  return a / b;
}

SH_HD int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Sequence b of the batch: its new tokens are rows row0 .. row0 + n - 1, at
// positions len - n + i (below 0 for i < n - len: rows that see nothing).
struct PagedSeq {
  int row0, n, len;
};

SH_HD PagedSeq paged_seq(int start, int end, int length, int tokens, int capacity) {
  PagedSeq s;
  s.row0 = clamp_int(start, 0, tokens);
  s.n = clamp_int(end, s.row0, tokens) - s.row0;
  s.len = clamp_int(length, 0, capacity);
  return s;
}

// The page of a position's table entry, or -1 where it is no page of the pool.
SH_HD int paged_page(int entry, int num_pages) { return entry >= 0 && entry < num_pages ? entry : -1; }

// ---- division of an attention call ----------------------------------------------
//
// A sequence's new tokens are taken in tiles of `per_tile` tokens, each with all
// query heads of one KV head. Laid end to end, in the order (sequence, KV head,
// tile), the tiles form a line on which a tile is as long as what it costs: the
// positions it may see and a fixed part. The line is cut into equal pieces, one
// per workgroup, so that every workgroup has the same to do whatever the lengths
// are; a tile cut by a piece's end is divided between workgroups at a multiple of
// `unit` positions, and its parts are merged. The cost of a sequence's first t
// tiles has a closed form, so a workgroup finds its piece by itself.

struct PagedPlan {
  const int *starts, *lengths;
  int batch, tokens, kv_heads, capacity;
  int per_tile;       // tokens of a tile
  int unit;           // positions of a unit: a tile is cut at multiples of it
  int window, sinks;  // window 0: none
  int workers;
  int min_piece;      // shortest piece of the line
  int whole_below;    // tiles of at most this cost are not cut
};

constexpr int kTileFixedCost = 64;  // of a tile, in positions
// Sums saturate here, far above any call's (starts out of order could pass 2^63).
constexpr long long kMaxLine = 1LL << 61;

SH_HD PagedSeq plan_seq(const PagedPlan &p, int b) {
  return paged_seq(p.starts[b], p.starts[b + 1], p.lengths[b], p.tokens, p.capacity);
}

SH_HD int plan_tiles(const PagedPlan &p, const PagedSeq &s) { return (s.n + p.per_tile - 1) / p.per_tile; }

// Cost of the sequence's first t tiles: tile i sees up to c + (i + 1) per_tile
// positions, or with a window no more than sinks + window + per_tile.
SH_HD long long plan_prefix(const PagedPlan &p, const PagedSeq &s, int t) {
  const long long c = s.len > s.n ? s.len - s.n : 0, R = p.per_tile;
  long long m = t, cap = 0;
  if (p.window > 0) {
    const int sinks = p.sinks < s.len ? p.sinks : s.len;
    cap = (long long)sinks + p.window + R;
    m = cap > c ? plan_div(cap - c, R) : 0;
    m = m < t ? m : t;
  }
  return (long long)t * kTileFixedCost + m * c + R * m * (m + 1) / 2 + (t - m) * cap;
}

SH_HD long long plan_add(long long a, long long b) { return a + b < kMaxLine ? a + b : kMaxLine; }

// Cost of a sequence (each KV head's tiles).
SH_HD long long plan_cost(const PagedPlan &p, const PagedSeq &s) {
  return plan_prefix(p, s, plan_tiles(p, s)) * p.kv_heads;
}

SH_HD long long plan_piece(const PagedPlan &p, long long total) {
  const long long q = plan_div(total + p.workers - 1, p.workers);
  return q > p.min_piece ? q : p.min_piece;
}

// A tile and where it lies on the line.
struct PagedTile {
  PagedSeq seq;
  int b, kv_head, tile;
  long long begin, cost;
};

// The tile that point x < prefix[parts] of the line lies in. prefix[i]: cost of
// the sequences before i * per (parts + 1 ascending values, prefix[0] = 0).
SH_HD PagedTile plan_locate(const PagedPlan &p, const long long *prefix, int parts, int per, long long x) {
  int lo = 0, hi = parts;  // prefix[lo] <= x < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (prefix[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  PagedTile t;
  long long at = prefix[lo];
  const int end = (lo + 1) * per < p.batch ? (lo + 1) * per : p.batch;
  t.b = lo * per < end ? lo * per : end - 1;
  t.seq = plan_seq(p, t.b);
  long long cost = plan_cost(p, t.seq);
  while (x >= at + cost && t.b + 1 < end) {
    at += cost;
    t.seq = plan_seq(p, ++t.b);
    cost = plan_cost(p, t.seq);
  }
  const int tiles = plan_tiles(p, t.seq);
  const long long one = plan_prefix(p, t.seq, tiles);  // a KV head's
  long long in = x - at;
  const long long head = one > 0 ? plan_div(in, one) : 0;
  t.kv_head = (int)(head < p.kv_heads ? head : p.kv_heads - 1);
  at += one * t.kv_head;
  in = x - at;
  int a = 0, z = tiles > 1 ? tiles : 1;  // prefix(a) <= in < prefix(z)
  while (z - a > 1) {
    const int mid = a + (z - a) / 2;
    if (plan_prefix(p, t.seq, mid) <= in)
      a = mid;
    else
      z = mid;
  }
  t.tile = a;
  t.begin = at + plan_prefix(p, t.seq, a);
  t.cost = plan_prefix(p, t.seq, a + 1) - plan_prefix(p, t.seq, a);
  return t;
}

// What a tile's tokens see: tokens first .. first + count - 1 of the sequence, the
// last at position hi - 1; positions [0, sinks) and [lo, hi), by units: unit j
// starts at position unit * (j + (j >= sink_units ? gap : 0)).
struct TileSpan {
  int first, count;
  int pos0;          // position of the first token (may be below 0)
  int lo, hi, sinks;
  int units, sink_units, gap;
};

SH_HD TileSpan plan_span(const PagedPlan &p, const PagedTile &t) {
  TileSpan s;
  s.first = t.tile * p.per_tile;
  s.count = t.seq.n - s.first < p.per_tile ? t.seq.n - s.first : p.per_tile;
  s.count = s.count > 0 ? s.count : 0;
  s.pos0 = t.seq.len - t.seq.n + s.first;
  s.hi = s.pos0 + s.count > 0 ? s.pos0 + s.count : 0;
  s.lo = 0;
  s.sinks = 0;
  s.gap = 0;
  s.sink_units = 0;
  s.units = (s.hi + p.unit - 1) / p.unit;
  if (p.window > 0) {
    const long long lo = (long long)s.pos0 - p.window + 1;
    s.lo = lo > 0 ? (int)lo : 0;
    s.sinks = p.sinks < s.hi ? p.sinks : s.hi;
    const int su = (s.sinks + p.unit - 1) / p.unit, wu = s.lo / p.unit;
    if (wu > su) {
      s.sink_units = su;
      s.gap = wu - su;
      s.units -= s.gap;
    }
  }
  return s;
}

// First position of unit j.
SH_HD int span_position(const TileSpan &s, int unit, int j) {
  return unit * (j + (j >= s.sink_units ? s.gap : 0));
}

// Units of a tile before point x of its cost: what a cut there leaves on its left.
SH_HD int plan_cut(const PagedPlan &p, const PagedTile &t, int units, long long x) {
  const long long in = x <= t.begin ? 0 : x >= t.begin + t.cost ? t.cost : x - t.begin;
  if (in == t.cost) return units;
  if (t.cost <= p.whole_below) return 2 * in >= t.cost ? units : 0;
  return (int)plan_div(in * units, t.cost);
}

// The cut of tile t by a piece that starts or ends strictly inside it: whether a
// point k * piece within the tile divides its units, from the first such point on.
struct TileParts {
  int first, count;  // pieces that touch the tile; count 1: not cut
};
SH_HD TileParts plan_parts(const PagedPlan &p, const PagedTile &t, int units, long long piece) {
  TileParts r;
  r.first = (int)plan_div(t.begin, piece);
  const int last = (int)plan_div(t.begin + t.cost - 1, piece);
  r.count = 1;
  for (int w = r.first + 1; w <= last; w++) {
    const int u = plan_cut(p, t, units, (long long)w * piece);
    if (u > 0 && u < units) r.count = last - r.first + 1;
    if (u > 0) break;  // (cuts ascend: one inside comes before any at the end)
  }
  return r;
}

// What a workgroup whose piece starts inside a cut tile leaves for the merge: the
// tile's rows and where its parts are. parts 0: nothing.
struct MergeItem {
  int parts, first_worker, first_slot;  // slot of the first part; worker w's others: 2 w
  int row0, tokens, kv_head;            // first token's row of q / out
};

// Worker w's step at point x of its piece [x0, x1): the tile there, the units of
// it that are the worker's and where they go. The next step is at tile.begin +
// tile.cost. A worker has two slots: 2 w for a tile that its piece starts in, 2 w +
// 1 for one that its piece ends in.
struct PieceStep {
  PagedTile tile;
  TileSpan span;
  int u0, u1;
  int slot;      // -1: the whole tile, to the output
  bool run;      // false: nothing of the tile is this worker's
  bool more;     // false: sums that saturated, the walk ends
};

SH_HD PieceStep plan_step(const PagedPlan &p, const long long *prefix, int parts, int per, long long piece,
                          int worker, long long x0, long long x1, long long x, MergeItem *item) {
  PieceStep r;
  r.tile = plan_locate(p, prefix, parts, per, x);
  r.more = x < r.tile.begin + r.tile.cost;
  r.span = plan_span(p, r.tile);
  const TileParts c = plan_parts(p, r.tile, r.span.units, piece);
  r.u0 = plan_cut(p, r.tile, r.span.units, x0);
  r.u1 = plan_cut(p, r.tile, r.span.units, x1);
  r.slot = -1;
  r.run = false;
  if (r.span.count == 0) return r;  // (no tile: only where sums saturated)
  if (c.count > 1) {
    r.slot = 2 * worker + (r.tile.begin > x0 ? 1 : 0);
    r.run = true;  // (of no units, too: the merge reads every part)
    if (r.tile.begin < x0 && worker == c.first + 1) {
      item->parts = c.count;
      item->first_worker = c.first;
      item->first_slot = 2 * c.first + (r.tile.begin > (long long)c.first * piece ? 1 : 0);
      item->row0 = r.tile.seq.row0 + r.span.first;
      item->tokens = r.span.count;
      item->kv_head = r.tile.kv_head;
    }
  } else {
    r.run = r.span.units > 0 ? r.u0 < r.u1 : worker == c.first;
  }
  return r;
}

// ---- argument checks that need no device -------------------------------------------

// nullptr, or what is wrong with the cache's sizes.
inline const char *check_paged_sizes(const sh_paged_kv *kv, int tokens, int heads) {
  if (!kv) return "the paged cache is NULL";
  if (kv->batch < 0 || kv->batch > kMaxPagedBatch) return "batch must be 0..65536";
  if (tokens < 0 || tokens > kMaxPagedTokens) return "tokens must be 0..2^22";
  if (kv->kv_heads < 1 || kv->kv_heads > kMaxPagedKvHeads) return "kv_heads must be 1..1024";
  if (heads < 1 || heads % kv->kv_heads != 0 || heads / kv->kv_heads > 128)
    return "heads must be kv_heads times 1..128";
  if (kv->head_dim < 1) return "head_dim must be positive";
  if (kv->page_size < 16 || kv->page_size > 65536 || (kv->page_size & (kv->page_size - 1)))
    return "page_size must be a power of two, 16..65536";
  if (kv->num_pages < 1) return "num_pages must be positive";
  if (kv->max_pages < 1 || kv->max_pages > kMaxPagedPositions / kv->page_size)
    return "max_pages must be positive and max_pages * page_size at most 2^28";
  return nullptr;
}

inline bool paged_dim_built(int head_dim) { return head_dim == 64 || head_dim == 128; }

inline size_t paged_pool_bytes(const sh_paged_kv *kv) {
  return (size_t)kv->num_pages * kv->kv_heads * kv->page_size * kv->head_dim * 2;
}

// The same of sh_pages_copy.
inline const char *check_pages_copy(int planes, size_t plane_stride, int num_pages, size_t page_bytes,
                                    int count) {
  if (planes < 0 || planes > 65535) return "planes must be 0..65535";
  if (num_pages < 1) return "num_pages must be positive";
  if (count < 0 || count > num_pages) return "count must be 0..num_pages";
  if (page_bytes < 16 || page_bytes % 16 != 0 || page_bytes > ((size_t)1 << 31))
    return "page_bytes must be a multiple of 16, at most 2^31";
  if (plane_stride % 16 != 0) return "plane_stride must be a multiple of 16";
  if (plane_stride < (size_t)num_pages * page_bytes && planes > 1)
    return "plane_stride must be at least num_pages * page_bytes";
  if (planes > 1 && plane_stride > ((size_t)1 << 62) / (size_t)planes) return "the pools exceed 2^62 bytes";
  return nullptr;
}

inline bool ranges_overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

}  // namespace sh
