// Packed attention: the launch of a call.  Host side only; not part of the C-ABI.
#pragma once
#include "attention_params.h"

namespace vfa {

int compute_units();

constexpr int kTileWaves = 4, kTileRows = 32 * kTileWaves, kStepRows = 16;

struct AttentionPlan {
  bool step;
  int rows;            // of a tile
  int64_t grid, join;  // workgroups; 0: no split
  int64_t line;        // step: units that a line may hold, counted in 32 bits
};

// The launch of a call, from its sizes alone: the lengths are on the device.  Measured as one side
// and the other, us, head dimension 128, 32 heads over 8 key heads unless said otherwise:
//   tiles of 16 rows up to 16 rows a sequence and, where two for each sequence and key head are fewer
//   than the CUs, up to 32 (8 sequences of 4000 keys, 32 rows: 33 against 40 in tiles of 128; 64
//   rows: 45, 40; 100 of 300 keys, 18 rows, 12 heads over 2: 21, 15; 64 of 500 keys, 32 rows: 54, 28);
//   up to 16 rows their even parts serve lengths that differ (32 of 2000 keys: 48, 53), at 8 % of
//   the time of 64 equal ones (1000 keys: 53, 46);
//   keys split for tiles of 16 above 768 and 512 a sequence, below which the second launch costs more
//   (one sequence of 600: 13.6 split, 12.2 whole; 1500: 13.9, 19.4; 3000: 14.5, 31; 8 of 500: 14.0,
//   11.5; 8 of 1000: 16.5 both);
//   for tiles of 128 where these number less than three quarters of the CUs (509 tokens after 2000
//   over 8 heads: 28 split, 57 whole; 2000 tokens over 16 heads, 240 tiles: 56, 49), in chunks of at
//   least 512 keys (400 tokens over 8 heads in chunks of 256: 18, whole 14).
// They see rows and sequences, not lengths, and cost most where these differ most: one sequence of 60000
// keys among 127 of one key, too few rows for a split, 664 (with 20000 rows of room, split, 126); 64
// sequences that share 32768 rows, not split, 541; 77 keys 7.8 in a room of 768 rows and 10.4, split, in
// one of 8192.  One kernel serves the whole call: 200 single tokens over 500 keys 108 and a prompt of
// 500 17, in one call 153, in tiles of 16; 100 over 1000 keys 93 and a prompt of 2000 56, in one call
// 137, in tiles of 128.
inline AttentionPlan attention_plan(AttentionParams& p) {
  const int64_t cus = compute_units();
  AttentionPlan plan{};
  auto shape = [&](bool step) {
    plan.step = step;
    plan.rows = step ? kStepRows : kTileRows;
    p.heads_per_tile = p.group < plan.rows ? p.group : plan.rows;
    p.parts = (p.group + p.heads_per_tile - 1) / p.heads_per_tile;
    p.head_blocks = p.heads / p.group * p.parts;
    p.tile_tokens = plan.rows / p.heads_per_tile;
  };
  shape(false);
  const int64_t rows = (int64_t)p.tokens * (p.group < kStepRows ? p.group : kStepRows);
  if (rows <= kStepRows * p.batch || (rows <= 2 * kStepRows * p.batch && 2 * p.batch * p.head_blocks < cus)) shape(true);
  // Divisions by these two as products: exact below 2^31 and 2^9.
  p.tile_shift = 31;
  while ((1 << (p.tile_shift - 31)) < p.tile_tokens) ++p.tile_shift;
  p.tile_mul = (uint32_t)(((uint64_t(1) << p.tile_shift) + p.tile_tokens - 1) / p.tile_tokens);
  p.row_mul = (65536 + p.heads_per_tile - 1) / p.heads_per_tile;
  // At most a tile per token, or whole tiles and one partial tile per sequence.
  const int64_t whole = p.tokens / p.tile_tokens;
  int64_t tiles = whole + p.batch + 2;
  if (tiles > p.tokens) tiles = p.tokens;
  if (plan.step) {
    // A CU holds one workgroup of dimension 128, two of 64.
    const bool split = p.keys > 768 && p.keys > 512 * p.batch;
    p.unit_shift = split ? 7 : 31;
    auto bound = [&] { return tiles * p.head_blocks * (((int64_t)p.keys >> p.unit_shift) + 1); };
    while (bound() >= int64_t(1) << 30 && p.unit_shift < 31) ++p.unit_shift;  // the kernel counts in 32 bits
    const int64_t units = bound();
    plan.line = p.head_blocks % 8 ? units : units / 8;
    plan.grid = (cus + 7) / 8 * 8 * (p.dim <= 64 ? 2 : 1);
    if (units < plan.grid) plan.grid = (units + 7) / 8 * 8;
    plan.join = split;
    p.slots = split ? 2 * plan.grid : 0;
    return plan;
  }
  // About how many tiles there are: whole ones, or one a sequence.
  int64_t about = p.batch < p.tokens ? p.batch : p.tokens;
  if (about < whole) about = whole;
  p.target = (int)(3 * cus);  // what the GPU holds of them
  p.min_chunk = 8;
  if (((int64_t)p.keys + 63) / 64 <= p.min_chunk || 4 * about * p.head_blocks >= 3 * cus) p.target = 0;
  p.slots = p.target ? 2 * p.target + p.head_blocks : 0;
  plan.join = p.target ? tiles * p.head_blocks : 0;
  plan.grid = tiles * p.head_blocks + (p.target ? p.slots : 0);
  plan.grid = (plan.grid + 7) / 8 * 8;  // whole rounds of the XCDs
  return plan;
}

}  // namespace vfa
