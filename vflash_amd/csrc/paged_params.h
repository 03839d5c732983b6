// Kernel-side parameter blocks of the rotary positions and the append to a paged cache (not part of the C-ABI).
#pragma once
#include "attention_params.h"

namespace vfa {

struct RotaryParams {
  const uint64_t* phases;  // [pairs], turns a position in 2^-64; null: no rotation
  const int64_t* axis;     // [pairs] in [0, axes); or null
  const int64_t* positions;  // [tokens][axes]; null: the tokens' own in their sequences
  int axes, pairs, interleaved;
  float magnitude;
};

struct RotateParams {
  const uint16_t *q, *k, *v;  // element (token, head, d) at token * *_ts + head * *_hs + d
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  uint16_t *q_out, *k_out;  // contiguous; q_out null: no q
  int64_t tokens, batch;
  int heads, key_heads, dim, f16;
  const int64_t* q_offsets;  // [batch + 1], or null: one token a sequence
  RotaryParams rotary;
  PagedCacheParams cache;  // values null: k goes to k_out, and there is no v
};

}  // namespace vfa
