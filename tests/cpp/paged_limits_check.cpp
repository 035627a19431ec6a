// Host check of the paged operators' argument checks at their largest sizes
// (strict_amd/csrc/paged.h).
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "paged.h"

using namespace sh;

static long long failures = 0;
#define CHECK(x)                                               \
  do {                                                         \
    if (!(x)) {                                                \
      if (failures++ < 20) std::printf("line %d: %s\n", __LINE__, #x); \
    }                                                          \
  } while (0)

static sh_paged_kv sizes(int num_pages, int kv_heads, int page_size, int head_dim) {
  sh_paged_kv kv;
  std::memset(&kv, 0, sizeof kv);
  kv.batch = 1, kv.max_pages = 1;
  kv.num_pages = num_pages, kv.kv_heads = kv_heads, kv.page_size = page_size, kv.head_dim = head_dim;
  return kv;
}

static void pools() {
  const auto refused = [](const sh_paged_kv &kv) { return check_paged_sizes(&kv, 1, kv.kv_heads) != nullptr; };
  // products that come round past 64 bits: to nothing, and to one page
  CHECK(refused(sizes(1 << 30, 1024, 65536, 128)));
  CHECK(refused(sizes((1 << 30) + 1, 1024, 65536, 128)));
  CHECK(refused(sizes(INT32_MAX, 1024, 65536, 128)) && refused(sizes(INT32_MAX, 1024, 65536, INT32_MAX)));
  // 2^62 bytes, and a page more
  CHECK(!refused(sizes(1 << 28, 1024, 65536, 128)) && refused(sizes((1 << 28) + 1, 1024, 65536, 128)));
  CHECK(!refused(sizes(1 << 29, 1024, 65536, 64)) && refused(sizes((1 << 29) + 1, 1024, 65536, 64)));
  // what is accepted is what is checked against the allocation
  for (int shift = 0; shift <= 30; shift++)
    for (int kv_heads : {1, 3, 8, 1024})
      for (int page_size : {16, 64, 65536})
        for (int head_dim : {64, 128}) {
          const sh_paged_kv kv = sizes(1 << shift, kv_heads, page_size, head_dim);
          const unsigned __int128 bytes = (unsigned __int128)kv.num_pages * kv_heads * page_size * head_dim * 2;
          CHECK(refused(kv) == (bytes > ((unsigned __int128)1 << 62)));
          if (!refused(kv)) CHECK(paged_pool_bytes(&kv) == bytes);
        }
}

static void thetas() {
  sh_paged_kv kv = sizes(4, 1, 65536, 128);
  kv.max_pages = 1 << 12;  // 2^28 positions
  CHECK(!check_rope_theta(&kv, kMaxPagedTokens, 1.0f) && !check_rope_theta(&kv, 1, 1e6f) && !check_rope_theta(&kv, 1, 3.4e38f));
  for (float theta : {0.0f, -1.0f, INFINITY, NAN, -0.0f}) CHECK(check_rope_theta(&kv, 1, theta));
  // (2^28 positions: frequencies of up to 2)
  CHECK(!check_rope_theta(&kv, 1, 0.5f) && check_rope_theta(&kv, 1, 0.25f) && check_rope_theta(&kv, 1, 1e-45f));
  for (int head_dim : {64, 128})
    for (int log2 = 1; log2 <= 149; log2++) {  // theta = 2^-log2: 2^(log2 (1 - 2 / head_dim)) times the positions
      kv.head_dim = head_dim, kv.page_size = 16, kv.max_pages = 1;
      const double exponent = log2 * (1.0 - 2.0 / head_dim);
      CHECK((check_rope_theta(&kv, 1, std::ldexp(1.0f, -log2)) != nullptr) == (exponent + 4 > 29));
      CHECK((check_rope_theta(&kv, 1 << 10, std::ldexp(1.0f, -log2)) != nullptr) == (exponent + 10 > 29));
    }
}

int main() {
  pools();
  thetas();
  std::printf("failures=%lld\n", failures);
  return failures == 0 ? 0 : 1;
}
