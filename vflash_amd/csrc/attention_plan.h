// Packed attention: the launch of a call.  Host side only; not part of the C-ABI.
#pragma once
#include "attention_params.h"

namespace vfa {

int compute_units();

constexpr int kTileWaves = 4, kTileRows = 32 * kTileWaves, kStepRows = 16;

struct AttentionPlan {
  bool step;
  int rows;            // of a tile
  int64_t grid, join;  // workgroups; 0: no split (step: 1, and 2 for small workgroups of the join)
  int waves;           // paged: of a workgroup
  int64_t line;        // step: units that a line may hold, counted in 32 bits
};

// The shape of the tiles.
inline void attention_shape(AttentionParams& p, AttentionPlan& plan, bool step) {
  plan.step = step;
  plan.rows = step ? kStepRows : kTileRows;
  p.heads_per_tile = p.group < plan.rows ? p.group : plan.rows;
  p.parts = (p.group + p.heads_per_tile - 1) / p.heads_per_tile;
  p.head_blocks = p.heads / p.group * p.parts;
  p.tile_tokens = plan.rows / p.heads_per_tile;
  // Divisions by these two as products: exact below 2^31 and 2^9.
  p.tile_shift = 31;
  while ((1 << (p.tile_shift - 31)) < p.tile_tokens) ++p.tile_shift;
  p.tile_mul = (uint32_t)(((uint64_t(1) << p.tile_shift) + p.tile_tokens - 1) / p.tile_tokens);
  p.row_mul = (65536 + p.heads_per_tile - 1) / p.heads_per_tile;
}

// At most a tile per token, or whole tiles and one partial tile per sequence.
inline int64_t attention_tiles_at_most(const AttentionParams& p) {
  const int64_t tiles = p.tokens / p.tile_tokens + p.batch + 2;
  return tiles < p.tokens ? tiles : p.tokens;
}

// The rest of the plan of tiles of 16; `per_cu`: workgroups that a CU holds.
inline void attention_step_plan(AttentionParams& p, AttentionPlan& plan, bool split, int per_cu) {
  const int64_t tiles = attention_tiles_at_most(p);
  p.unit_shift = split ? 7 : 31;
  auto bound = [&] { return tiles * p.head_blocks * (((int64_t)p.keys >> p.unit_shift) + 1); };
  while (bound() >= int64_t(1) << 30 && p.unit_shift < 31) ++p.unit_shift;  // the kernel counts in 32 bits
  const int64_t units = bound();
  plan.line = p.head_blocks % 8 ? units : units / 8;
  plan.grid = (compute_units() + 7) / 8 * 8 * per_cu;
  if (units < plan.grid) plan.grid = (units + 7) / 8 * 8;
  plan.join = split;
  p.slots = split ? 2 * plan.grid : 0;
}

// The rest of the plan of tiles of 128.
inline void attention_tiles_plan(AttentionParams& p, AttentionPlan& plan) {
  const int64_t cus = compute_units();
  const int64_t tiles = attention_tiles_at_most(p), whole = p.tokens / p.tile_tokens;
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
}

// Tiles of 16 rows, or of 128.
inline bool attention_few_rows(const AttentionParams& p) {
  const int64_t rows = (int64_t)p.tokens * (p.group < kStepRows ? p.group : kStepRows);
  return rows <= kStepRows * p.batch || (rows <= 2 * kStepRows * p.batch && 2 * p.batch * p.head_blocks < compute_units());
}

// Over a paged cache, in tiles of 16 or 128 as packed attention is.  For tiles of 16 a sequence's room stands for its
// length, which varies: the keys are split from 768 where the tiles leave half of the workgroups idle, and else from
// 1536.  Equal lengths that fill their room, us whole and split, 32 heads over 8 of dimension 128 in bf16 and E4M3, and of 64 in bf16: one of
// 500 keys 11.4 12.0, 10.2 11.4, 8.1 10.4; of 1000 16.3 12.3, 14.5 11.8, 10.7 10.9; of 2000 25.9 13.5, 22.7 12.9, 16.2
// 11.9; 16 of 1000 18.6 21.5, 15.6 18.2, 11.9 15.6; 16 of 2000 33.0 34.7, 24.4 22.0, 17.8 19.7; 32 of 2000 51.9 54.5,
// 29.9 34.5, 27.0 31.5.  E4M3 tiles take half the LDS, and two workgroups where bf16 has one: 61 sequences of 1 to 8191
// keys 117 us, 129 with one.
inline AttentionPlan paged_attention_plan(AttentionParams& p, bool e4m3) {
  AttentionPlan plan{};
  attention_shape(p, plan, true);
  // About how many tiles of 16 there are: whole ones, or one a sequence.
  int64_t tiles = p.batch < p.tokens ? p.batch : p.tokens;
  if (tiles < p.tokens / p.tile_tokens) tiles = p.tokens / p.tile_tokens;
  tiles *= p.head_blocks;
  // Beside the few rows of packed attention, drafts and short pieces whose tiles of 16 are so few that reading K and V
  // again for each costs less than the long chain of a tile of 128.  us in tiles of 16 and of 128: bf16, 8 query heads a key
  // head, 1 sequence of 500 keys, 5 tokens 11.5 16.0, 4 of 2000 15.5 24.9, of 8000 22.6 28.3, 16 of 2000, 12 tokens (96 tiles)
  // 28.3 26.9; 100 keys 8.3 7.5; E4M3, 32 heads over 8, 16 of 2000 keys, 16 tokens 42.7 45.7, 8 of 1000, 64 tokens 31.2 43.1, 128
  // tokens (2048 tiles) 60.8 54.5, 8 of 4000, 24 tokens 48.9 46.5; up to 64 rows of 128 at any length, 16 of 8000, 9 tokens 97 145.
  attention_shape(p, plan, false);
  const bool few = attention_few_rows(p);
  const bool drafts = (int64_t)p.tokens * p.group <= 64 * p.batch;
  const bool pieces = e4m3 ? tiles <= 4 * compute_units() && (drafts || tiles * p.keys <= 1 << 20)
                           : 2 * tiles <= compute_units() && tiles * p.keys <= 163840 && p.keys > 128;
  if (!few && !pieces) {
    attention_tiles_plan(p, plan);
    return plan;
  }
  attention_shape(p, plan, true);
  const int per_cu = (p.dim <= 64 ? 2 : 1) * (e4m3 ? 2 : 1);
  const int64_t held = (int64_t)compute_units() * per_cu;
  const bool split = p.keys > (2 * tiles < held ? 768 : 1536);
  // More whole sequences than the GPU holds go in workgroups of two waves, twice as many: 128 of 250 keys in bf16 32 us, in
  // four waves 42; of 700 70 and 75; 64 of 250 in E4M3, which fit, 13.2 and 12.7.
  plan.waves = !split && tiles > held ? 2 : 4;
  // More than twice as many, of little room, in workgroups of one wave: 86 of up to 32 keys, 56 heads of their own, in bf16
  // 21 us, of two waves 50; of 250 93 and 108; of 500, of one with two slots, 174 and 170.  120 of 32, 8 key heads, 8.7, 13.1.
  if (!split && tiles > 2 * held && p.keys <= 256) plan.waves = 1;
  attention_step_plan(p, plan, split, plan.waves == 1 ? (p.dim <= 64 ? 16 : 8) : per_cu * 4 / plan.waves);
  // Of several tokens a sequence a workgroup takes two units at least, half as many segments for their join: four tokens after
  // 8000 keys in E4M3 18.6 us, by single units 22.0, after 2000 14.3 either way; one token of 2000 keys 14.4 and 13.7.
  p.least_units = split && p.tokens > p.batch ? 2 : 1;
  if (plan.join) {
    // A join of 256 threads takes 16 / rows segments of a tile at a time, one of 1024 four times as many, but its
    // grid takes longer to start: 128 sequences of 1000 keys in E4M3 58 and 62 us, 15 of four tokens 25.8 and 23.1.
    const int64_t each = (p.tokens + p.batch) / (p.batch + 1);
    int64_t rows = 1;
    while (rows < 16 && rows < each * p.heads_per_tile) rows *= 2;
    if (plan.grid * rows <= 64 * tiles) plan.join = 2;
  }
  return plan;
}

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
  AttentionPlan plan{};
  attention_shape(p, plan, false);
  if (attention_few_rows(p)) attention_shape(p, plan, true);
  if (plan.step) {
    attention_step_plan(p, plan, p.keys > 768 && p.keys > 512 * p.batch, p.dim <= 64 ? 2 : 1);
    return plan;
  }
  attention_tiles_plan(p, plan);
  return plan;
}

}  // namespace vfa
