// Host check of find_tile (strict_amd/csrc/paged.h): for starts in any order each tile of each
// sequence is found once, at a number below the total, and behind the last there is none.
#include <algorithm>
#include <array>
#include <climits>
#include <cstdio>
#include <random>
#include <set>
#include <vector>

#include "paged.h"

using namespace sh;

static long long failures = 0;
#define CHECK(x)                                               \
  do {                                                         \
    if (!(x)) {                                                \
      if (failures++ < 20) std::printf("line %d: %s\n", __LINE__, #x); \
    }                                                          \
  } while (0)

struct HostWave {
  typedef std::array<int, 64> Int;
  template <class F>
  static Int each(F f) {
    Int v;
    for (int i = 0; i < 64; i++) v[i] = f(i);
    return v;
  }
  template <class F>
  static Int map(const Int &x, F f) {
    return each([&](int i) { return f(x[i]); });
  }
  static Int scan(Int v) {
    for (int i = 1; i < 64; i++) {
      CHECK((long long)v[i] + v[i - 1] <= INT_MAX);
      v[i] = std::min(v[i] + v[i - 1], kMaxTiles);
    }
    return v;
  }
  static int read(const Int &v, int lane) {
    CHECK(lane >= 0 && lane < 64);
    return v[lane & 63];
  }
  template <class F>
  static uint64_t ballot(const Int &v, F f) {
    uint64_t those = 0;
    for (int i = 0; i < 64; i++) those |= (uint64_t)(f(v[i]) ? 1 : 0) << i;
    return those;
  }
  static int nth(uint64_t those, int n) {
    CHECK(n >= 0 && n < __builtin_popcountll(those));
    for (; n > 0; n--) those &= those - 1;
    return __builtin_ctzll(those);
  }
};

int main() {
  std::mt19937 rng(5);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  const int sizes[] = {1, 63, 64, 65, 128, 129, 700, 4096};
  long long cases = 0;
  for (int round = 0; round < 240; round++) {
    PagedPlan p = {};
    p.batch = round % 3 == 0 ? sizes[upto(7)] : 1 + upto(round % 3 == 1 ? 70 : 300);
    p.per_tile = 1 + upto(round % 2 ? 127 : 15);
    const int kind = round % 5;  // in order; any numbers; some out of order; all rows again and again; none
    std::vector<int> starts(p.batch + 1);
    int at = upto(3);
    for (int &s : starts) {
      s = kind == 1 ? (int)rng() : kind == 4 ? 7 : at;
      at += upto(9) == 0 ? upto(p.batch > 1000 ? 60 : 600) : upto(3);
    }
    p.tokens = kind == 1 ? upto(3000) : std::max(starts[p.batch], 7) + upto(2);
    if (kind == 2)
      for (int i = upto(5); i >= 0; i--) starts[upto(p.batch)] = upto(p.tokens + 50) - 20;
    if (kind == 3) {
      p.tokens = std::min(p.tokens, 40);
      for (int b = 0; b <= p.batch; b++) starts[b] = b % 2 ? p.tokens : 0;
    }
    p.starts = starts.data();
    std::vector<int> lengths(p.batch, 0);
    p.lengths = lengths.data();
    p.capacity = 1;
    std::set<std::pair<int, int>> left;
    for (int b = 0; b < p.batch; b++) {
      CHECK(plan_tiles_of(p, b) == plan_tiles(p, plan_seq(p, b)));
      for (int t = 0; t < plan_tiles(p, plan_seq(p, b)); t++) left.insert({b, t});
    }
    const int all = (int)left.size();
    CHECK(kind != 0 || all <= p.batch + p.tokens / p.per_tile);
    int last_back = INT_MAX, last_b = -1;
    for (int i = 0; i < all; i++) {
      int back = -1, total = -1;
      const int b = find_tile<HostWave>(p, i, &back, &total);
      CHECK(total == all);
      CHECK(b >= 0 && b < p.batch && back >= 0);
      if (b < 0 || b >= p.batch) break;
      const int tile = plan_tiles(p, plan_seq(p, b)) - 1 - back;
      CHECK(tile >= 0);
      CHECK(left.erase({b, tile}) == 1);
      if (p.batch > 64) CHECK(b >= last_b);
      if (p.batch <= 64) CHECK(i == 0 || back >= last_back);
      last_back = back;
      last_b = b;
    }
    CHECK(left.empty());
    for (int i : {all, all + 1, all + 32768, kMaxTiles}) {
      int back = 0, total = -1;
      CHECK(find_tile<HostWave>(p, i, &back, &total) == -1);
      CHECK(total == all);
    }
    cases++;
  }
  {  // more tiles than there are numbers: those there are, and an end
    PagedPlan p = {};
    p.batch = 4096;
    p.per_tile = 1;
    p.tokens = kMaxPagedTokens;
    std::vector<int> starts(p.batch + 1);
    for (int b = 0; b <= p.batch; b++) starts[b] = b % 2 ? p.tokens : 0;
    p.starts = starts.data();
    for (int i : {0, 1, p.tokens - 1, p.tokens, 1 << 29, kMaxTiles - 1}) {
      int back = 0, total = 0;
      CHECK(find_tile<HostWave>(p, i, &back, &total) == 2 * (i / p.tokens) && back == i % p.tokens && total == kMaxTiles);
    }
    int back = 0, total = 0;
    CHECK(find_tile<HostWave>(p, kMaxTiles, &back, &total) == -1);
  }
  std::printf("cases=%lld failures=%lld\n", cases, failures);
  return failures == 0 ? 0 : 1;
}
