// The argument checks of sh_sample_f32 and sh_adjust_logits_* that need no device.
#pragma once

#include <cstddef>
#include <cstdint>

#include "strict_hip.h"

namespace sh {

constexpr int kMaxSampleN = 1 << 20;
constexpr int kMaxSampleRows = 1 << 16;
constexpr int kMaxRuleTokens = 1 << 29;

// nullptr, or what is wrong.
inline const char *check_sample_sizes(int rows, int n, int ld) {
  if (rows < 0 || rows > kMaxSampleRows) return "rows must be 0..65536";
  if (n < 1 || n > kMaxSampleN) return "n must be 1..2^20";
  if (ld < n) return "ld must be at least n";
  return nullptr;
}

inline const char *check_logits_sizes(int rows, int n, int ldx, int ldy, const sh_logit_rules *r) {
  if (const char *wrong = check_sample_sizes(rows, n, ldx)) return wrong;
  if (ldy < n) return "ldy must be at least n";
  if (r->tokens && !r->lengths) return "tokens need lengths";
  if (r->tokens && (r->max_tokens < 0 || r->max_tokens > kMaxRuleTokens)) return "max_tokens must be 0..2^29";
  if (r->bias_starts && r->bias_count < 0) return "bias_count must not be negative";
  if (r->bias_starts && r->bias_count > 0 && (!r->bias_tokens || !r->bias_values))
    return "bias_starts needs bias_tokens and bias_values";
  if (r->masks && (!r->mask_of || r->num_masks < 1)) return "masks need mask_of and num_masks";
  return nullptr;
}

}  // namespace sh
