// A KV cache in pages: which rows and positions a batch's sequences have, how
// the attention over them is divided among workgroups, and the argument checks
// of the paged operators that need no device. Plain C++ on host and device, so
// that the bounds below are checked on the CPU for any device data (tests/cpp).
//
// What lies in device memory (starts, lengths, page table) cannot be checked on
// the host: every value is brought into its range here before it indexes
// anything, and a page number out of range makes its positions invisible.
#pragma once

#include <cmath>
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
constexpr double kMaxPoolBytes = 4611686018427387904.0;  // 2^62: sizes and ends of pools in 64 bits

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
  int unit;           // positions of a unit, a power of two: a tile is cut at multiples of it
  int unit_shift;     // its logarithm
  int window, sinks;  // window 0: none
  int workers;
  double inv_workers; // 1 / workers
  int min_piece;      // shortest piece of the line
  int whole_below;    // tiles of at most this cost are not cut
};

constexpr int kTileFixedCost = 64;  // of a tile, in positions
// Places on the line are whole numbers below 2^53 in fp64, of which every operation
// below is exact and one instruction (of a 64-bit integer product or comparison it
// takes several, of a division some hundred: planning took 5 us of a kernel with
// those). The line of a call is at most kMaxLine (check_paged_sizes); sums over starts
// out of order, which may count tokens twice, stop there.
typedef double Line;
constexpr Line kMaxLine = 4503599627370496.0;  // 2^52

// floor(a / b): exact, as a quotient that rounds to a whole number it is below
// differs from it by less than 1 / a of it.
SH_HD Line plan_div(Line a, Line b) { return floor(a / b); }

SH_HD PagedSeq plan_seq(const PagedPlan &p, int b) {
  return paged_seq(p.starts[b], p.starts[b + 1], p.lengths[b], p.tokens, p.capacity);
}

SH_HD int plan_tiles(const PagedPlan &p, const PagedSeq &s) { return (s.n + p.per_tile - 1) / p.per_tile; }

// Cost of the sequence's first t tiles: tile i sees up to c + (i + 1) per_tile
// positions, or with a window no more than sinks + window + per_tile.
SH_HD Line plan_prefix(const PagedPlan &p, const PagedSeq &s, int t) {
  const Line c = s.len > s.n ? s.len - s.n : 0, R = p.per_tile;
  Line m = t, cap = 0;
  if (p.window > 0) {
    const int sinks = p.sinks < s.len ? p.sinks : s.len;
    cap = (Line)sinks + p.window + R;
    m = cap > c ? plan_div(cap - c, R) : 0;
    m = m < t ? m : t;
  }
  return t * (Line)kTileFixedCost + m * c + R * m * (m + 1) * 0.5 + (t - m) * cap;
}

SH_HD Line plan_add(Line a, Line b) { return a + b < kMaxLine ? a + b : kMaxLine; }

// A sequence on the line: its tiles, and what one KV head's cost together.
struct PlanSeq {
  PagedSeq seq;
  int tiles;
  Line one;
};

SH_HD PlanSeq plan_sequence(const PagedPlan &p, int b) {
  PlanSeq s;
  s.seq = plan_seq(p, b);
  s.tiles = plan_tiles(p, s.seq);
  s.one = plan_prefix(p, s.seq, s.tiles);
  return s;
}

// The cost of the sequence's last tile, its largest.
SH_HD Line plan_last(const PagedPlan &p, const PlanSeq &s) {
  return s.tiles > 1 ? s.one - plan_prefix(p, s.seq, s.tiles - 1) : s.one;
}

// (At least total / workers, with room for the roundings.) A piece that is somewhat
// shorter than the largest tile becomes as long: most tiles then fit one and need no
// merge. Of 392 tiles of about one cost over 512 workers: 87 -> 73 us a call. From 3/8 of it on,
// 8 sequences of up to 333 tokens: 35 -> 46, 4 of up to 512 65 -> 86.
SH_HD Line plan_piece(const PagedPlan &p, Line total, Line largest) {
  const Line q = floor(total * p.inv_workers) + 2;
  const Line r = q < largest && 8 * q >= 5 * largest ? largest : q;
  return r > p.min_piece ? r : p.min_piece;
}

// Workers for a call: `most`, or fewer where even full tables would not give each of
// them a shortest piece. A multiple of 8.
inline int plan_workers(int batch, int kv_heads, int tokens, int capacity, int per_tile, int min_piece, int most) {
  const double tiles = (double)tokens / per_tile + batch;  // at most, of each KV head
  const double line = tiles * kv_heads * ((double)capacity + per_tile + kTileFixedCost);
  const double n = line / min_piece + 8;
  return n < most ? ((int)n + 7) / 8 * 8 : most;
}

// A tile and where it lies on the line.
struct PagedTile {
  PagedSeq seq;
  int b, kv_head, tile;
  Line begin, cost;
};

// The last i < parts with prefix[i] <= x (prefix ascends from 0).
SH_HD int plan_find(const Line *prefix, int parts, Line x) {
  int lo = 0, hi = parts;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (prefix[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The tile that point x of the line lies in. at: cost of the sequences before part *
// per, of which `s` is the first (plan_part_first), the sequence of x among the `per`
// from there on.
SH_HD int plan_part_first(const PagedPlan &p, int part, int per) {
  const int end = (part + 1) * per < p.batch ? (part + 1) * per : p.batch;
  return part * per < end ? part * per : end - 1;
}
SH_HD PagedTile plan_locate(const PagedPlan &p, PlanSeq s, int part, int per, Line at, Line x) {
  PagedTile t;
  const int end = (part + 1) * per < p.batch ? (part + 1) * per : p.batch;
  t.b = plan_part_first(p, part, per);
  while (x >= at + s.one * p.kv_heads && t.b + 1 < end) {
    at += s.one * p.kv_heads;
    s = plan_sequence(p, ++t.b);
  }
  t.seq = s.seq;
  const Line head = p.kv_heads > 1 && s.one > 0 ? plan_div(x - at, s.one) : 0;
  t.kv_head = head < p.kv_heads ? (int)head : p.kv_heads - 1;
  at += s.one * t.kv_head;
  int a = 0, z = s.tiles > 1 ? s.tiles : 1;  // prefix(a) <= x - at < prefix(z)
  while (z - a > 1) {
    const int mid = a + (z - a) / 2;
    if (plan_prefix(p, t.seq, mid) <= x - at)
      a = mid;
    else
      z = mid;
  }
  t.tile = a;
  const Line before = a > 0 ? plan_prefix(p, t.seq, a) : 0;
  t.begin = at + before;
  t.cost = (s.tiles > 1 ? plan_prefix(p, t.seq, a + 1) : s.one) - before;
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
  s.units = (s.hi + p.unit - 1) >> p.unit_shift;
  if (p.window > 0) {
    const long long lo = (long long)s.pos0 - p.window + 1;
    s.lo = lo > 0 ? (int)lo : 0;
    s.sinks = p.sinks < s.hi ? p.sinks : s.hi;
    const int su = (s.sinks + p.unit - 1) >> p.unit_shift, wu = s.lo >> p.unit_shift;
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
SH_HD int plan_cut(const PagedPlan &p, const PagedTile &t, int units, Line x) {
  if (x <= t.begin) return 0;
  if (x >= t.begin + t.cost) return units;
  const Line in = x - t.begin;
  if (t.cost <= p.whole_below) return 2 * in >= t.cost ? units : 0;
  return (int)plan_div(in * units, t.cost);
}

// What a workgroup whose piece starts inside a cut tile leaves for the merge: the
// tile's rows and where its parts are. parts 0: nothing.
struct MergeItem {
  int parts, first_worker, first_slot;  // slot of the first part; worker w's others: 2 w
  int row0, tokens, kv_head;            // first token's row of q / out
};

// Worker w's step at point x of its piece [x0, x1), x0 = w * piece: the tile there,
// the units of it that are the worker's and where they go. The next step is at
// tile.begin + tile.cost. A tile is cut if two pieces' ends lie in it, or one that
// divides its units. A worker has two slots: 2 w for a cut tile that its piece
// starts in (or with), 2 w + 1 for one that its piece ends in.
struct PieceStep {
  PagedTile tile;
  TileSpan span;
  int u0, u1;
  int slot;   // -1: the whole tile, to the output
  bool run;   // false: nothing of the tile is this worker's
  bool more;  // false: sums that saturated, the walk ends
};

// The first worker of a tile.
SH_HD int plan_first(const PagedTile &t, int worker, Line piece, Line x0) {
  return t.begin >= x0 ? worker : worker - (int)plan_div(x0 - t.begin + piece - 1, piece);
}

SH_HD PieceStep plan_step(const PagedPlan &p, const PagedTile &t, Line piece, int worker, Line x0, Line x,
                          MergeItem *item) {
  PieceStep r;
  r.tile = t;
  r.span = plan_span(p, t);
  const Line end = t.begin + t.cost;
  r.more = x < end;
  r.u0 = plan_cut(p, t, r.span.units, x0);
  r.u1 = plan_cut(p, t, r.span.units, x0 + piece);
  r.slot = -1;
  r.run = false;
  if (r.span.count == 0) return r;  // (no tile: only where sums saturated)
  const bool left = t.begin < x0, right = end > x0 + piece;
  bool cut = left && (right || t.begin < x0 - piece);
  cut = cut || (right && end > x0 + 2 * piece);
  cut = cut || (left && r.u0 > 0 && r.u0 < r.span.units) || (right && r.u1 > 0 && r.u1 < r.span.units);
  if (cut) {
    r.slot = 2 * worker + (t.begin > x0 ? 1 : 0);
    r.run = true;  // (of no units, too: the merge reads every part)
    if (left && t.begin >= x0 - piece) {
      item->first_worker = worker - 1;
      item->parts = 2 + (right ? (int)plan_div(end - x0 - 1, piece) : 0);
      item->first_slot = 2 * (worker - 1) + (t.begin > x0 - piece ? 1 : 0);
      item->row0 = t.seq.row0 + r.span.first;
      item->tokens = r.span.count;
      item->kv_head = t.kv_head;
    }
  } else {
    r.run = r.span.units > 0 ? r.u0 < r.u1 : !left;
  }
  return r;
}

// ---- a workgroup a tile -------------------------------------------------------------
//
// Calls whose tiles are not cut: the tiles of all sequences are numbered through, and a
// workgroup finds the one of its number by itself, a wave looking at 64 numbers at once.
// W is that wave: each(f) and map(v, f) have f of each lane (and its value), scan the sums
// of lanes 0 .. own, at most kMaxTiles, read the value of a lane, ballot the lanes whose
// value f takes, nth the n-th of such lanes (on the device registers and lane moves; on the
// host arrays, so that the search is checked there for any starts).
constexpr int kMaxWholeBatch = 4096;
constexpr int kMaxTiles = (1 << 30) - 1;  // (two such sums fit an int)

SH_HD int plan_tiles_of(const PagedPlan &p, int b) {
  const int from = clamp_int(p.starts[b], 0, p.tokens), end = clamp_int(p.starts[b + 1], from, p.tokens);
  return (end - from + p.per_tile - 1) / p.per_tile;
}

// The sequence of tile `at` (0 or more), how many of its tiles come behind that, and how
// many tiles there are in all; -1: fewer than that. The longest come first: of up to 64 sequences the
// last tile of each, then the last but one, and so on; of more, up to kMaxWholeBatch,
// sequence by sequence. (Sequences whose starts are out of order may have more tiles together
// than all tokens make.)
template <class W>
SH_HD int find_tile(const PagedPlan &p, int at, int *back, int *total) {
  typedef typename W::Int Int;
  const int per = (p.batch + 63) / 64;
  if (per == 1) {
    const Int mine = W::each([&](int lane) { return lane < p.batch ? plan_tiles_of(p, lane) : 0; });
    // tiles with fewer than n behind them
    const auto behind = [&](int n) { return W::read(W::scan(W::map(mine, [&](int t) { return t < n ? t : n; })), 63); };
    int n = 0, end = p.tokens / p.per_tile + 1;  // behind(n) <= at < behind(end): no sequence has more tiles than that
    *total = behind(end);
    if (*total <= at) return -1;
    while (end - n > 1) {
      const int mid = (n + end) / 2;
      if (behind(mid) <= at)
        n = mid;
      else
        end = mid;
    }
    *back = n;
    const int which = at - behind(n);
    return W::nth(W::ballot(mine, [&](int t) { return t > n; }), which);
  }
  int first = 0;
  for (int step = per;; step = 1) {  // a 64th of the sequences in each lane, then one
    const Int up_to = W::scan(W::each([&](int lane) {
      int sum = 0;
      for (int i = 0; i < step; i++) {
        const int b = first + lane * step + i;
        if (b < p.batch && (step == per || lane < per)) {
          sum += plan_tiles_of(p, b);
          sum = sum < kMaxTiles ? sum : kMaxTiles;
        }
      }
      return sum;
    }));
    if (step == per) *total = W::read(up_to, 63);
    const uint64_t before = W::ballot(up_to, [&](int t) { return t <= at; });
    if (before == ~(uint64_t)0) return -1;
    const int lane = __builtin_popcountll(before);  // (sums ascend)
    at -= lane == 0 ? 0 : W::read(up_to, lane - 1);
    first += lane * step;
    if (step == 1) break;
  }
  *back = at;
  return first;
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
  // (what an attention call may cost: kMaxLine, in tiles of one token)
  if (((double)tokens + kv->batch) * kv->kv_heads * ((double)kv->max_pages * kv->page_size + 512.0) > kMaxLine)
    return "(tokens + batch) * kv_heads * (max_pages * page_size + 512) exceeds 2^52";
  // (exact in fp64 for the head sizes there are: 31 and 10 bits, and powers of two)
  if ((double)kv->num_pages * kv->kv_heads * kv->page_size * kv->head_dim * 2.0 > kMaxPoolBytes)
    return "num_pages * kv_heads * page_size * head_dim exceeds 2^61 (a pool of 2^62 bytes)";
  return nullptr;
}

// RoPE's angles, position * theta^(-2i / head_dim) in fp64, are to be below 2^29: there
// a step of fp64 is 2^-24, fp32's of their cosines, and the quadrant fits an int.
// Positions reach from -tokens to the capacity; with theta >= 1 no frequency exceeds 1.
inline const char *check_rope_theta(const sh_paged_kv *kv, int tokens, float theta) {
  if (!(theta > 0.0f) || !std::isfinite(theta)) return "theta must be positive and finite";
  const double capacity = (double)kv->max_pages * kv->page_size, reach = capacity > tokens ? capacity : tokens;
  const double fastest = theta < 1.0f ? std::pow((double)theta, -(kv->head_dim - 2.0) / kv->head_dim) : 1.0;
  if (reach * fastest > 536870912.0)
    return "theta: max_pages * page_size (or tokens) * theta^(-(head_dim - 2) / head_dim) exceeds 2^29";
  return nullptr;
}

// RoPE's frequencies, theta^(-2i / head_dim) for i < head_dim / 2: a power each, as a product
// of two powers is another value, and the angles of far positions then steps of fp32 off.
inline void rope_frequencies(float theta, int head_dim, double *freq) {
  for (int i = 0; i < head_dim / 2; i++) freq[i] = std::pow((double)theta, -2.0 * i / head_dim);
}

inline bool paged_dim_built(int head_dim) { return head_dim == 64 || head_dim == 128; }

inline size_t paged_pool_bytes(const sh_paged_kv *kv) {
  return (size_t)kv->num_pages * kv->kv_heads * kv->page_size * kv->head_dim * 2;
}

// ---- pages of 8-bit values ------------------------------------------------------------
//
// A page: k [kv_heads][page_size][head_dim], v alike, then their scales
// [2][kv_heads][page_size], a byte each, so that a copy of a page takes all of it. A
// multiple of 32 bytes, as page_size is one of 16.
inline size_t paged8_page_bytes(const sh_paged_kv8 *kv) {
  return (size_t)kv->kv_heads * kv->page_size * 2 * ((size_t)kv->head_dim + 1);
}
// (Of sizes that check_paged_sizes takes: at most 1 + 1 / head_dim times 2^62 bytes.)
inline size_t paged8_pool_bytes(const sh_paged_kv8 *kv) { return (size_t)kv->num_pages * paged8_page_bytes(kv); }

// The cache's sizes and index tensors as those of one of 16-bit values without pools.
inline sh_paged_kv paged8_index(const sh_paged_kv8 *kv) {
  sh_paged_kv i = {nullptr,   nullptr,       kv->page_table, kv->lengths,   kv->starts,  kv->batch,
                   kv->max_pages, kv->num_pages, kv->page_size,  kv->kv_heads, kv->head_dim};
  return i;
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
