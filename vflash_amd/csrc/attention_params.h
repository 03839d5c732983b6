// Kernel-side parameter block of packed attention (not part of the C-ABI).
#pragma once
#include <stdint.h>

namespace vfa {

struct AttentionParams {
  const uint16_t *q, *k, *v;  // element (row, head, d) at row * *_ts + head * *_hs + d
  uint16_t* out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  const int64_t *q_offsets, *k_offsets, *k_lengths;  // k_lengths: or null
  int tokens, keys;  // rows
  int64_t batch;
  int heads, group, dim;  // group: query heads of a key head
  int causal;
  float c;  // scale * log2(e)
  float shift, bound;  // of bf16 weights: attention_shift, attention_bound
  // The tiles' shape.
  int heads_per_tile;  // of a key head's group; a group of more than the tile's rows has `parts` blocks
  int parts, head_blocks;
  int tile_tokens;
  uint32_t tile_mul;  // x / tile_tokens = x * tile_mul >> tile_shift
  int tile_shift, row_mul;  // r / heads_per_tile = r * row_mul >> 16
  // Splitting of the keys, off where target is 0.
  int target, min_chunk;  // items, blocks of 64 keys
  int64_t slots;          // what the workspace holds
  int unit_shift;  // attention_step: log2 of a unit's keys (31: a whole sequence)
  float* part;  // [slot][row][d], then [slot][row] maxima and sums
  float* part_ml;
};

}  // namespace vfa
