// Host check of strict_amd/csrc/paged.h: that the pieces of an attention call cover
// every unit of every tile once, that what is written for the merge is what it
// reads, and that nothing indexes out of range whatever the device data are; and of
// the argument checks of the paged operators and of sampling.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "paged.h"
#include "sample.h"

using namespace sh;

static long long failures = 0;
#define CHECK(x)                                               \
  do {                                                         \
    if (!(x)) {                                                \
      if (failures++ < 20) std::printf("line %d: %s\n", __LINE__, #x); \
    }                                                          \
  } while (0)

static constexpr int kParts = 256;

static std::vector<Line> prefix_of(const PagedPlan &p, int per, Line *largest) {
  *largest = 0;
  std::vector<Line> prefix(kParts + 1, 0);
  for (int t = 0; t < kParts; t++) {
    Line sum = 0;
    for (int b = t * per; b < (t + 1) * per && b < p.batch; b++) {
      const PlanSeq s = plan_sequence(p, b);
      sum = plan_add(sum, s.one * p.kv_heads);
      for (int i = 0; i < s.tiles && i < 50; i++)
        CHECK(plan_prefix(p, s.seq, i + 1) - plan_prefix(p, s.seq, i) <= plan_last(p, s));
      *largest = std::max(*largest, plan_last(p, s));
    }
    prefix[t + 1] = plan_add(prefix[t], sum);
  }
  return prefix;
}

struct Written {
  std::vector<std::pair<int, int>> units;  // of whoever took a range of the tile
  int direct = 0;
  std::set<int> slots;
};

// orderly: starts ascend, so that every tile is there once.
static void walk(const PagedPlan &p, bool orderly, int group) {
  const int per = (p.batch + kParts - 1) / kParts;
  Line largest;
  const std::vector<Line> prefix = prefix_of(p, per, &largest);
  const Line total = prefix[kParts], piece = plan_piece(p, total, largest);
  CHECK(piece * p.workers >= total);
  // the workers that the host gives a call with these sizes have room for it, too
  PagedPlan q = p;
  q.workers = plan_workers(p.batch, p.kv_heads, p.tokens, p.capacity, p.per_tile, p.min_piece, 768);
  q.inv_workers = 1.0 / q.workers;
  CHECK(q.workers > 0 && q.workers <= 768 && q.workers % 8 == 0 && plan_piece(q, total, largest) * q.workers >= total);
  std::map<std::tuple<int, int, int>, Written> tiles;
  std::vector<MergeItem> items(p.workers);
  std::map<int, std::tuple<int, int, int>> slot_owner;
  for (int w = 0; w < p.workers; w++) {
    MergeItem item = {0, 0, 0, 0, 0, 0};
    const Line x0 = w * piece, x1 = x0 + piece < total ? x0 + piece : total;
    long long steps = 0;
    for (Line x = x0; x < x1;) {
      const int part = plan_find(prefix.data(), kParts, x);
      const PagedTile tile = plan_locate(p, plan_sequence(p, plan_part_first(p, part, per)), part, per, prefix[part], x);
      const PieceStep s = plan_step(p, tile, piece, w, x0, x, &item);
      if (orderly) CHECK(plan_first(tile, w, piece, x0) == (int)std::floor(tile.begin / piece));
      CHECK(s.tile.b >= 0 && s.tile.b < p.batch);
      CHECK(s.tile.kv_head >= 0 && s.tile.kv_head < p.kv_heads);
      CHECK(s.span.count >= 0 && s.span.count <= p.per_tile);
      CHECK(s.tile.seq.row0 + s.span.first + s.span.count <= p.tokens);
      CHECK(s.span.units >= 0 && s.u0 >= 0 && s.u0 <= s.u1 && s.u1 <= s.span.units);
      CHECK(s.span.hi <= p.capacity);
      if (s.span.units > 0) {
        CHECK(span_position(s.span, p.unit, s.span.units - 1) < s.span.hi);
        CHECK(span_position(s.span, p.unit, s.span.units - 1) + p.unit >= s.span.hi);
      }
      if (!s.more) {
        CHECK(!orderly);
        break;
      }
      CHECK(s.tile.begin <= x && x < s.tile.begin + s.tile.cost);
      if (s.run) {
        CHECK(s.slot < 2 * p.workers);
        Written &t = tiles[std::make_tuple(s.tile.b, s.tile.kv_head, s.tile.tile)];
        if (s.slot < 0) {
          t.direct++;
          t.units.push_back({0, s.span.units});
          CHECK(s.u0 == 0 && s.u1 == s.span.units);
        } else {
          t.units.push_back({s.u0, s.u1});
          t.slots.insert(s.slot);
          if (orderly) {
            CHECK(slot_owner.count(s.slot) == 0);
            slot_owner[s.slot] = std::make_tuple(s.tile.b, s.tile.kv_head, s.tile.tile);
          }
        }
      }
      x = s.tile.begin + s.tile.cost;
      if (++steps > 10000000) {
        CHECK(!"walk ends");
        break;
      }
    }
    items[w] = item;
  }
  if (!orderly) return;
  std::map<std::tuple<int, int>, const MergeItem *> merged;  // by (first row, KV head)
  for (const MergeItem &it : items)
    if (it.parts > 0) {
      CHECK(merged.count(std::make_tuple(it.row0, it.kv_head)) == 0);
      merged[std::make_tuple(it.row0, it.kv_head)] = &it;
    }
  size_t there = 0, cut = 0;
  for (int b = 0; b < p.batch; b++) {
    const PagedSeq s = plan_seq(p, b);
    for (int h = 0; h < p.kv_heads; h++)
      for (int t = 0; t < plan_tiles(p, s); t++, there++) {
        const auto at = tiles.find(std::make_tuple(b, h, t));
        CHECK(at != tiles.end());
        if (at == tiles.end()) continue;
        PagedTile tile;
        tile.seq = s;
        tile.tile = t;
        const TileSpan span = plan_span(p, tile);
        // every position that a token sees lies in a unit
        for (int i = 0; i < span.count; i++) {
          const int pos = span.pos0 + i;
          for (int k : {0, p.sinks - 1, pos - p.window + 1, pos / 2, pos}) {
            if (k < 0 || k > pos || k >= s.len) continue;
            if (p.window > 0 && !(k > pos - p.window || k < p.sinks)) continue;
            int found = 0;
            for (int u = 0; u < span.units; u++) {
              const int p0 = span_position(span, p.unit, u);
              found += p0 <= k && k < p0 + p.unit;
            }
            CHECK(found == 1);
          }
        }
        const Written &w = at->second;
        int next = 0;
        for (const auto &u : w.units) {  // workers ascend
          CHECK(u.first == next);
          next = u.second;
        }
        CHECK(next == span.units);
        const auto m = merged.find(std::make_tuple(s.row0 + span.first, h));
        if (w.direct) {
          CHECK(w.direct == 1 && w.units.size() == 1 && m == merged.end());
        } else {
          cut++;
          CHECK(m != merged.end());
          if (m == merged.end()) continue;
          const MergeItem &it = *m->second;
          std::set<int> reads;
          for (int j = 0; j < it.parts; j++) reads.insert(j == 0 ? it.first_slot : 2 * (it.first_worker + j));
          CHECK(reads == w.slots);
          CHECK(it.tokens == span.count);
        }
      }
  }
  CHECK(there == tiles.size());
  CHECK(cut == merged.size());
  (void)group;
}

int main() {
  std::mt19937 rng(7);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  long long cases = 0;
  for (int round = 0; round < 1500; round++) {
    PagedPlan p;
    const bool orderly = round % 4 != 3;
    p.batch = 1 + (round % 11 == 0 ? upto(900) : upto(20));
    p.kv_heads = 1 + upto(5);
    p.capacity = 16 << upto(9);
    const int group = 1 + upto(round % 5 == 0 ? 127 : 15);
    const int rows = group > 16 ? 128 : (round & 1) ? 16 : 128;
    p.per_tile = rows / group;
    p.unit_shift = 6 + upto(2);
    p.unit = 1 << p.unit_shift;
    p.window = round % 3 == 0 ? 1 + upto(p.capacity) : 0;
    p.sinks = upto(round % 2 ? 8 : p.capacity);
    p.workers = 8 * (1 + upto(99));
    p.inv_workers = 1.0 / p.workers;
    p.min_piece = 64 << upto(3);
    p.whole_below = round % 2 ? 0 : upto(2000);
    std::vector<int> starts(p.batch + 1), lengths(p.batch);
    int at = upto(3);
    for (int b = 0; b <= p.batch; b++) {
      starts[b] = orderly ? at : (int)rng();
      at += round % 7 == 0 ? upto(1) : upto(4) == 0 ? upto(400) : upto(3);
    }
    p.tokens = orderly ? starts[p.batch] + upto(2) : upto(3000);
    for (int &l : lengths) l = orderly ? upto(p.capacity) + (upto(9) == 0 ? 5 : 0) : (int)rng();
    p.starts = starts.data();
    p.lengths = lengths.data();
    walk(p, orderly, group);
    cases++;
  }
  {  // the largest sizes, out of order: sums saturate and every walk still ends
    PagedPlan p;
    p.batch = 4096;
    p.tokens = kMaxPagedTokens;
    p.kv_heads = 1;
    p.capacity = kMaxPagedPositions;
    p.per_tile = 1;
    p.unit = 64;
    p.unit_shift = 6;
    p.window = p.sinks = 0;
    p.workers = 64;
    p.inv_workers = 1.0 / 64;
    p.min_piece = 256;
    p.whole_below = 0;
    std::vector<int> starts(p.batch + 1), lengths(p.batch, kMaxPagedPositions);
    for (int b = 0; b <= p.batch; b++) starts[b] = b % 2 ? p.tokens : 0;
    p.starts = starts.data();
    p.lengths = lengths.data();
    const int per = (p.batch + kParts - 1) / kParts;
    Line largest;
    const std::vector<Line> prefix = prefix_of(p, per, &largest);
    CHECK(prefix[kParts] == kMaxLine);
    for (int t = 0; t < kParts; t++) CHECK(prefix[t] <= prefix[t + 1]);
    const Line piece = plan_piece(p, prefix[kParts], largest);
    for (int w = 0; w < p.workers; w++) {
      MergeItem item = {0, 0, 0, 0, 0, 0};
      const int part = plan_find(prefix.data(), kParts, w * piece);
      const PagedTile tile = plan_locate(p, plan_sequence(p, plan_part_first(p, part, per)), part, per, prefix[part], w * piece);
      const PieceStep s = plan_step(p, tile, piece, w, w * piece, w * piece, &item);
      CHECK(s.tile.b >= 0 && s.tile.b < p.batch && s.tile.kv_head < p.kv_heads);
      CHECK(s.u0 >= 0 && s.u1 <= s.span.units);
    }
  }
  // page numbers
  for (int n : {1, 7}) {
    CHECK(paged_page(-1, n) == -1 && paged_page(n, n) == -1 && paged_page(n - 1, n) == n - 1);
    CHECK(paged_page((int)0x80000000, n) == -1 && paged_page(0x7fffffff, n) == -1 && paged_page(0, n) == 0);
  }
  // refusals
  sh_paged_kv kv;
  std::memset(&kv, 0, sizeof kv);
  kv.batch = 2, kv.max_pages = 4, kv.num_pages = 9, kv.page_size = 16, kv.kv_heads = 2, kv.head_dim = 64;
  CHECK(!check_paged_sizes(&kv, 5, 4));
  CHECK(check_paged_sizes(nullptr, 5, 4));
  auto refused = [&](int sh_paged_kv::*field, int value) {
    sh_paged_kv bad = kv;
    bad.*field = value;
    return check_paged_sizes(&bad, 5, 4) != nullptr;
  };
  for (int v : {0, 8, 15, 17, 48, -16, 1 << 17}) CHECK(refused(&sh_paged_kv::page_size, v));
  for (int v : {16, 32, 65536}) CHECK(!refused(&sh_paged_kv::page_size, v));
  for (int v : {0, -1, 3, 4096}) CHECK(refused(&sh_paged_kv::kv_heads, v));
  for (int v : {0, -3, (1 << 24) + 1}) CHECK(refused(&sh_paged_kv::max_pages, v));
  {
    sh_paged_kv big = kv;
    big.max_pages = 1 << 24;
    big.kv_heads = 8;
    CHECK(check_paged_sizes(&big, kMaxPagedTokens, 8) && !check_paged_sizes(&big, 1 << 20, 8));
  }
  CHECK(!refused(&sh_paged_kv::max_pages, 1 << 24));
  for (int v : {0, -3}) CHECK(refused(&sh_paged_kv::num_pages, v));
  for (int v : {-1, kMaxPagedBatch + 1}) CHECK(refused(&sh_paged_kv::batch, v));
  CHECK(!refused(&sh_paged_kv::batch, 0));
  for (int v : {0, -64}) CHECK(refused(&sh_paged_kv::head_dim, v));
  for (int h : {0, -2, 3, 258}) CHECK(check_paged_sizes(&kv, 5, h));
  CHECK(!check_paged_sizes(&kv, 5, 256));
  CHECK(check_paged_sizes(&kv, -1, 4) && check_paged_sizes(&kv, kMaxPagedTokens + 1, 4));
  CHECK(paged_dim_built(64) && paged_dim_built(128) && !paged_dim_built(96) && !paged_dim_built(256));
  CHECK(!check_pages_copy(2, 160, 10, 16, 10) && !check_pages_copy(0, 0, 1, 16, 0) && !check_pages_copy(1, 0, 10, 16, 3));
  CHECK(check_pages_copy(-1, 160, 10, 16, 1) && check_pages_copy(2, 144, 10, 16, 1) && check_pages_copy(2, 168, 10, 16, 1));
  CHECK(check_pages_copy(2, 160, 0, 16, 0) && check_pages_copy(2, 160, 10, 8, 1) && check_pages_copy(2, 240, 10, 24, 1));
  CHECK(check_pages_copy(2, 160, 10, 16, 11) && check_pages_copy(2, 160, 10, 16, -1) && check_pages_copy(2, 160, 10, 0, 1));
  CHECK(check_pages_copy(65535, (size_t)1 << 60, 10, 16, 1));
  CHECK(!check_sample_sizes(0, 1, 1) && !check_sample_sizes(65536, 1 << 20, 1 << 20));
  CHECK(check_sample_sizes(-1, 5, 5) && check_sample_sizes(65537, 5, 5) && check_sample_sizes(1, 0, 5));
  CHECK(check_sample_sizes(1, (1 << 20) + 1, 1 << 21) && check_sample_sizes(1, 5, 4));
  char memory[64];
  CHECK(ranges_overlap(memory, 16, memory + 15, 4) && !ranges_overlap(memory, 16, memory + 16, 4));
  CHECK(ranges_overlap(memory + 4, 4, memory, 64) && !ranges_overlap(memory + 32, 4, memory, 32));
  std::printf("cases=%lld failures=%lld\n", cases, failures);
  return failures == 0 ? 0 : 1;
}
