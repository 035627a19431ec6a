// Host check of paged.h for calls whose tiles are not cut: every tile is one worker's, by
// all of its units, and no more of a walk indexes out of range, whatever the device data are.
#define main paged_check_main
#include "paged_check.cpp"
#undef main

static void walk_whole(const PagedPlan &p, bool orderly) {
  const int per = (p.batch + kParts - 1) / kParts;
  Line largest;
  const std::vector<Line> prefix = prefix_of(p, per, &largest);
  const Line total = prefix[kParts], piece = plan_piece(p, total, largest);
  CHECK(piece * p.workers >= total);
  std::map<std::tuple<int, int, int>, int> tiles;
  for (int w = 0; w < p.workers; w++) {
    const Line x0 = w * piece, x1 = x0 + piece < total ? x0 + piece : total;
    long long steps = 0;
    for (Line x = x0; x < x1;) {
      const int part = plan_find(prefix.data(), kParts, x);
      const PagedTile tile = plan_locate(p, plan_sequence(p, plan_part_first(p, part, per)), part, per, prefix[part], x);
      const PieceStep s = plan_step_whole(p, tile, x0, x);
      CHECK(s.tile.b >= 0 && s.tile.b < p.batch);
      CHECK(s.tile.kv_head >= 0 && s.tile.kv_head < p.kv_heads);
      CHECK(s.span.count >= 0 && s.span.count <= p.per_tile);
      CHECK(s.tile.seq.row0 + s.span.first + s.span.count <= p.tokens);
      CHECK(s.slot == -1 && s.u0 == 0 && s.u1 == s.span.units && s.span.units >= 0);
      CHECK(s.span.hi <= p.capacity);
      if (s.span.units > 0) CHECK(span_position(s.span, p.unit, s.span.units - 1) < s.span.hi);
      if (!s.more) {
        CHECK(!orderly);
        break;
      }
      if (s.run) tiles[std::make_tuple(s.tile.b, s.tile.kv_head, s.tile.tile)]++;
      x = s.tile.begin + s.tile.cost;
      if (++steps > 10000000) {
        CHECK(!"walk ends");
        break;
      }
    }
  }
  if (!orderly) return;
  size_t there = 0;
  for (int b = 0; b < p.batch; b++) there += (size_t)p.kv_heads * plan_tiles(p, plan_seq(p, b));
  CHECK(there == tiles.size());
  for (const auto &t : tiles) CHECK(t.second == 1);
}

int main() {
  std::mt19937 rng(5);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  long long cases = 0;
  for (int round = 0; round < 900; round++) {
    PagedPlan p;
    const bool orderly = round % 5 != 4;
    p.per_tile = 16 / (1 + upto(15));
    p.unit = round % 2 ? 64 : 128;
    p.unit_shift = round % 2 ? 6 : 7;
    p.min_piece = 64;
    p.whole_below = 192;
    p.batch = 1 + (round % 13 == 0 ? upto(700) : upto(12));
    p.kv_heads = 1 + upto(8);
    p.capacity = 16 * (1 + upto(8 * p.unit / 16 - 1));
    p.window = upto(1) ? 0 : 1 + upto(p.capacity + 40);
    p.sinks = upto(3) == 0 ? upto(p.capacity) : upto(70);
    std::vector<int> starts(p.batch + 1), lengths(p.batch);
    int at = upto(3);
    for (int b = 0; b <= p.batch; b++) {
      starts[b] = orderly ? at : (int)rng();
      at += upto(20) == 0 ? upto(700) : upto(std::max(1, p.per_tile));  // (more than the positions, too)
    }
    p.tokens = orderly ? starts[p.batch] + upto(2) : upto(3000);
    for (int &l : lengths) l = orderly ? upto(p.capacity) + (upto(9) == 0 ? 5 : 0) : (int)rng();
    p.starts = starts.data();
    p.lengths = lengths.data();
    p.workers = plan_workers(p.batch, p.kv_heads, p.tokens, p.capacity, p.per_tile,
                             p.capacity + p.per_tile + kTileFixedCost, 512);
    p.inv_workers = 1.0 / p.workers;
    walk_whole(p, orderly);
    cases++;
  }
  std::printf("cases=%lld failures=%lld\n", cases, failures);
  return failures == 0 ? 0 : 1;
}
