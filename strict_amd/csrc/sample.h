// The argument checks of sh_sample_f32 that need no device.
#pragma once

#include <cstddef>
#include <cstdint>

namespace sh {

constexpr int kMaxSampleN = 1 << 20;
constexpr int kMaxSampleRows = 1 << 16;

// nullptr, or what is wrong.
inline const char *check_sample_sizes(int rows, int n, int ld) {
  if (rows < 0 || rows > kMaxSampleRows) return "rows must be 0..65536";
  if (n < 1 || n > kMaxSampleN) return "n must be 1..2^20";
  if (ld < n) return "ld must be at least n";
  return nullptr;
}

}  // namespace sh
