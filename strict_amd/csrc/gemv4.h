// Matrices of 4-bit weights (sh_gemv_w4a16_*): their layout and the argument checks that
// need no device.
#pragma once

#include <cstddef>
#include <cstdint>

namespace sh {

constexpr int kMaxGemv4Batch = 64, kMaxGemv4N = 1 << 28, kMaxGemv4K = 1 << 24, kMaxGemv4Ldx = 1 << 25;

// The layout that the products read: tiles of 16 rows by 128 columns, columns first, as
// the matrix instructions take them: lane l's 16 bytes are row l % 16, dword j of them
// columns 32 j + 8 (l / 16) .. + 7, the first in the lowest bits (1 KiB a tile). Then the
// tiles' scales, 4 of each row (64 bytes a tile). Then a word for each 16 rows: bit r: row
// r has a scale of 255, a NaN; bits 16 and 17: scales with which some weight is no normal
// number of fp16, of bf16. Rows and columns that fill up a tile are zeros.
struct Gemv4Layout {
  size_t row_tiles, col_tiles;
  Gemv4Layout(int N, int K) : row_tiles(((size_t)N + 15) / 16), col_tiles(((size_t)K + 127) / 128) {}
  size_t scales_at() const { return row_tiles * col_tiles * 1024; }
  size_t flags_at() const { return row_tiles * col_tiles * 1088; }
  size_t bytes() const { return (flags_at() + row_tiles * 4 + 15) / 16 * 16; }
};

// nullptr, or what is wrong.
inline const char *check_e2m1_sizes(int N, int K) {
  if (N < 0 || N > kMaxGemv4N) return "N must be 0..2^28";
  if (K < 32 || K % 32 != 0 || K > kMaxGemv4K) return "K must be a multiple of 32, 32..2^24";
  return nullptr;
}
inline const char *check_gemv4_sizes(int batch, int K, int N, int ldx, int ldy) {
  if (batch < 1 || batch > kMaxGemv4Batch) return "batch must be 1..64";
  if (const char *wrong = check_e2m1_sizes(N, K)) return wrong;
  // (64 rows' bytes in 32 bits)
  if (ldx < K || ldx % 8 != 0 || ldx > kMaxGemv4Ldx) return "ldx must be a multiple of 8, at least K and at most 2^25";
  if (ldy < N) return "ldy must be at least N";
  return nullptr;
}

}  // namespace sh
