// Kernel-side parameter block of packed attention (not part of the C-ABI).
#pragma once
#include <stdint.h>

namespace vfa {

// Where keys and values lie: rows of two tensors, pages in the operands' type, pages of E4M3 codes.
enum AttentionStore { kStoreRows, kStorePages, kStoreE4M3 };

// A cache of pages: element (page, k or v, key head, slot, d), contiguous, in the operands' 16-bit type
// or, with scales, E4M3 codes and a binary32 factor of each (page, k or v, key head, slot).
struct PagedCacheParams {
  uint8_t* values;
  float* scales;  // or null
  int64_t pages;
  const int64_t* table;  // [batch][width], the page of keys slot * i .. slot * (i + 1) - 1
  int64_t width;
  const int64_t* lengths;  // [batch]
  int page_shift;          // log2 of a page's keys, 4 at least
  int key_heads;
};

struct AttentionParams {
  const uint16_t *q, *k, *v;  // element (row, head, d) at row * *_ts + head * *_hs + d
  uint16_t* out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
  const int64_t *q_offsets, *k_offsets, *k_lengths;  // k_lengths: or null
  int tokens, keys;  // rows; pages: the most that a sequence has
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
  // Of a call over pages, last: the loads of the others' arguments stay as wide as they are.
  PagedCacheParams cache;  // these instead of k, v, k_offsets and k_lengths; q_offsets may be null
  uint32_t least_units;    // of a workgroup
  int32_t* begun;          // [workgroup][4]: AttentionBegun
};

}  // namespace vfa
