// The host check of paged.h (paged_check.cpp, whose walk this is) with the 16-row tiles that
// the attention kernels over pages of 8-bit values take: units of 64 positions at head_dim
// 128 and of 128 at head_dim 64, where the shortest piece is half a unit.
#define main paged_check_main
#include "paged_check.cpp"
#undef main

int main() {
  std::mt19937 rng(12);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  long long cases = 0;
  for (int round = 0; round < 600; round++) {
    PagedPlan p;
    const bool orderly = round % 5 != 4;
    const int group = 1 + upto(15);
    p.per_tile = 16 / group;
    p.unit_shift = round % 3 == 0 ? 6 : 7;
    p.unit = 1 << p.unit_shift;
    p.min_piece = 64;
    p.whole_below = 192;
    p.batch = 1 + (round % 13 == 0 ? upto(700) : upto(12));
    p.kv_heads = 1 + upto(8);
    p.capacity = 16 << upto(round % 4 == 0 ? 12 : 8);
    p.window = round % 2 ? 0 : 1 + upto(p.capacity + 40);
    p.sinks = upto(3) == 0 ? upto(p.capacity) : upto(70);
    std::vector<int> starts(p.batch + 1), lengths(p.batch);
    int at = upto(3);
    for (int b = 0; b <= p.batch; b++) {
      starts[b] = orderly ? at : (int)rng();
      at += upto(std::max(1, p.per_tile));
    }
    p.tokens = orderly ? starts[p.batch] + upto(2) : upto(3000);
    for (int &l : lengths) l = orderly ? upto(p.capacity) + (upto(9) == 0 ? 5 : 0) : (int)rng();
    p.starts = starts.data();
    p.lengths = lengths.data();
    p.workers = plan_workers(p.batch, p.kv_heads, p.tokens, p.capacity, p.per_tile, p.min_piece, 512);
    p.inv_workers = 1.0 / p.workers;
    walk(p, orderly, group);
    cases++;
  }
  std::printf("cases=%lld failures=%lld\n", cases, failures);
  return failures == 0 ? 0 : 1;
}
