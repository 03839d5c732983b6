// Packed attention: what its kernels share.  Kernel-side only; not part of the C-ABI.
//
// Sequence s has nq queries, rows of q and out, and nk keys, rows of k and v.  Query head h
// reads key head h / group.  With the queries last in their sequence,
//
//   lim(i) = causal ? max(0, nk - nq + i + 1) : nk          the keys that query i sees
//   out(i) = sum_{j < lim} p_j v_j / sum_{j < lim} p_j,  p_j = 2^(c q_i . k_j - m),
//   c = scale log2(e), m any number near the largest exponent; out(i) = 0 where lim = 0.
//
// The exponent is one fused c s - c m, off by c m's rounding, the same factor for all of a row.
// Past kAttentionFar that rounding would overflow the factor; such rows take c (s - m).
//
// A tile is up to BQ (token, head) pairs of one sequence that read one key head, so grouped
// heads share what they load.  An item is a tile and a range of its keys; ranges of one tile
// leave an unnormalised sum each, which attention_join adds up.
#pragma once
#include "attention_params.h"
#include "common.h"

#include <type_traits>

namespace vfa {

typedef _Float16 v8hf __attribute__((ext_vector_type(8)));
typedef _Float16 v2hf __attribute__((ext_vector_type(2)));
typedef short v4s16 __attribute__((ext_vector_type(4)));

// Below every finite exponent: 2^(x - m) is 0 for a masked x = -inf, with no inf - inf.
#define VFA_LOWEST (-3.4028234663852886e38f)
// The running maximum follows the scores only once they pass it by 2^8, so that the sums are
// rarely rescaled; p is then at most 2^8 and, in binary16, carries 2^6 more, which keeps 30
// binary orders below the largest p out of the format's subnormals.
constexpr float kAttentionSlack = 8.0f;
constexpr float kAttentionFar = 4194304.0f;  // 2^22: a rounding of 1/4
template <bool F16>
constexpr float kAttentionShift = F16 ? 6.0f : 0.0f;

// 2^(c (s - m)) times 2^shift, m the row's maximum before its scaling.
template <bool F16, bool FAR>
__device__ __forceinline__ float attention_weight(float s, float c, float m, float ref) {
  return __builtin_amdgcn_exp2f(FAR ? (s - m) * c + kAttentionShift<F16> : __builtin_fmaf(s, c, ref));
}
// A row's maximum as its statistics carry it: scaled, and finite where it saw nothing.
__device__ __forceinline__ float attention_top(float m, float c) { return fmaxf(m * c, VFA_LOWEST); }

template <bool F16>
__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8hf, a), __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8hf, a), __builtin_bit_cast(v8hf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// Two values to the operand type, to nearest even.  Not pack_bf16x2: the values come from
// v_exp_f32, whose result the next instruction may not read yet, and the compiler places the wait
// states for its own instructions only.
template <bool F16>
__device__ __forceinline__ int pack2(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(int, v2hf{(_Float16)a, (_Float16)b});
  else return __builtin_bit_cast(int, v2bf{(__bf16)a, (__bf16)b});
}

// Eight bytes per lane, transposed inside each group of 16 lanes: lane 4 r + c of a group gives
// the address of elements 4 c .. 4 c + 3 of row r, and lane i receives element i of the four rows.
typedef int v2i __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2i lds_read_tr16(const uint8_t* p) {
  typedef __attribute__((address_space(3))) v4s16 lds_v4s16;
  return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s16*)(uint32_t)lds_addr(p)));
}

// Over the two half waves, and over the two 16-lane rows of each.
__device__ __forceinline__ float max_across32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_across16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------------------
// The schedule.  Lengths are known on the device alone, so every wave derives it again from the
// offsets: a prefix sum over the sequences, 64 at a time.  Two sequences without keys stand for
// the rows of q before the first offset and after the last, which are written as zeros.
// Offsets are clamped to the operands, so none leads outside them.

// Inclusive prefix sum over the wave; the total lands in every lane of `total`.
__device__ __forceinline__ int wave_scan(int v, int lane, int& total) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31);
  const int r2 = __builtin_amdgcn_readlane(v, 47), r3 = __builtin_amdgcn_readlane(v, 63);
  v += lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2;
  total = r0 + r1 + r2 + r3;
  return v;
}

struct AttentionSeq {
  int q0, k0, nq, nk;
};
// Sequence s of 0 .. batch + 1 (0 and batch + 1: the rows outside the offsets).
__device__ __forceinline__ AttentionSeq attention_sequence(const AttentionParams& p, int64_t s) {
  auto clamp = [](int64_t v, int lo, int hi) { return (int)(v < lo ? lo : v > hi ? hi : v); };
  AttentionSeq r{0, 0, 0, 0};
  if (s > p.batch + 1) return r;
  r.q0 = s == 0 ? 0 : clamp(p.q_offsets[s - 1], 0, p.tokens);
  r.nq = (s > p.batch ? p.tokens : clamp(p.q_offsets[s], r.q0, p.tokens)) - r.q0;
  if (s == 0 || s > p.batch) return r;
  r.k0 = clamp(p.k_offsets[s - 1], 0, p.keys);
  r.nk = p.k_lengths ? clamp(p.k_lengths[s - 1], 0, p.keys - r.k0) : clamp(p.k_offsets[s], r.k0, p.keys) - r.k0;
  return r;
}

struct AttentionItem {
  AttentionSeq seq;  // all uniform
  int tile, tiles;   // of the sequence
  int split, splits;
  int chunk;         // keys of a split
  int slot;          // of the tile's split 0, where it has several
  int head_block;
  bool live;
};

// The unit `index` of the launch: an item, or with JOIN a tile (all its splits).
template <bool JOIN>
__device__ __forceinline__ AttentionItem attention_item(const AttentionParams& p, uint32_t index) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t n = p.batch + 2;
  auto tiles_of = [&](const AttentionSeq& s) {
    return (int)(((uint32_t)s.nq + (uint32_t)p.tile_tokens - 1) / (uint32_t)p.tile_tokens);
  };
  auto blocks_of = [](const AttentionSeq& s) { return ((uint32_t)s.nk + 63) >> 6; };
  AttentionSeq mine{};
  // Keys of a split, in blocks of 64: the whole sequence where the tiles fill the GPU, else as
  // many as make about p.target items.
  uint32_t chunk = 1u << 25;
  int tiles = 0;
  if (p.target) {
    float work = 0;
    for (int64_t base = 0; base < n; base += 64) {
      mine = attention_sequence(p, base + lane);
      int t = tiles_of(mine), sum;
      wave_scan(t, lane, sum);
      tiles += sum;
      work += wave_sum((float)t * (float)blocks_of(mine));
    }
    work = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(work)));
    chunk = max((uint32_t)p.min_chunk, (uint32_t)fminf(ceilf(work * (float)p.head_blocks / (float)p.target), 33554432.0f));
  }
  auto splits_of = [&](const AttentionSeq& s) { return (int)max(1u, (blocks_of(s) + chunk - 1) / chunk); };
  auto slots_of = [](int t, int sp) { return sp > 1 ? t * sp : 0; };
  AttentionItem it{};
  // Units and slots per head block; the grid's order needs them before the search.  A split
  // sequence has more keys than a chunk, so the slots are at most 2 p.target.
  int units = 0, slots = 0;
  for (int64_t base = 0; base < n; base += 64) {
    if (!p.target || n > 64) mine = attention_sequence(p, base + lane);
    const int t = tiles_of(mine), sp = splits_of(mine);
    int sum;
    wave_scan(t * sp, lane, sum);
    units += sum;
    wave_scan(slots_of(t, sp), lane, sum);
    slots += sum;
  }
  if (p.target && (int64_t)slots * p.head_blocks > p.slots) {  // not reached: a bound on the memory
    chunk = 1u << 25;
    units = tiles;
  }
  int total = units;  // of what `index` counts
  if constexpr (JOIN) total = tiles;
  // Workgroup b runs on XCD b % 8.  Where the head blocks divide among the XCDs, each XCD
  // takes whole ones, one after another, so that its L2 holds their keys.
  int x;
  if (p.head_blocks % 8 == 0) {
    const int i = (int)(index >> 3);
    if (total == 0 || i >= total * (p.head_blocks / 8)) return it;
    it.head_block = (int)(index & 7) + 8 * (i / total);
    x = i % total;
  } else {
    it.head_block = (int)(index % (uint32_t)p.head_blocks);
    x = (int)(index / (uint32_t)p.head_blocks);
    if (x >= total) return it;
  }
  int before = 0, slots_before = 0;
  for (int64_t base = 0; base < n; base += 64) {
    if (n > 64) mine = attention_sequence(p, base + lane);
    const int t = tiles_of(mine), sp = splits_of(mine), own = JOIN ? t : t * sp;
    int sum, slot_sum;
    const int incl = wave_scan(own, lane, sum);
    const int slot_incl = wave_scan(slots_of(t, sp), lane, slot_sum);
    if (x < before + sum) {
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + incl > x));
      auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      it.seq = AttentionSeq{pick(mine.q0), pick(mine.k0), pick(mine.nq), pick(mine.nk)};
      it.tiles = pick(t);
      it.splits = pick(sp);
      const int in = x - before - pick(incl - own);
      const int back = JOIN ? in : in / it.splits;  // tiles from the last to the first: longest first
      it.split = JOIN ? 0 : in % it.splits;
      it.tile = it.tiles - 1 - back;
      it.chunk = (int)min((uint64_t)chunk * 64, (uint64_t)INT32_MAX);
      it.slot = it.head_block * slots + slots_before + pick(slot_incl - slots_of(t, sp)) + back * it.splits;
      it.live = true;
      return it;
    }
    before += sum;
    slots_before += slot_sum;
  }
  return it;
}

// Row r of a tile: its token in the sequence, its head, and whether it is one.
struct AttentionRow {
  int token, head;
  bool live;
};
__device__ __forceinline__ AttentionRow attention_row(const AttentionParams& p, const AttentionItem& it, int r) {
  const int in = (int)((uint32_t)r / (uint32_t)p.heads_per_tile);
  const int h = it.head_block % p.parts * p.heads_per_tile + r - in * p.heads_per_tile;
  AttentionRow row;
  row.token = it.tile * p.tile_tokens + in;
  row.head = it.head_block / p.parts * p.group + h;
  row.live = in < p.tile_tokens && row.token < it.seq.nq && h < p.group;
  return row;
}

// Keys that the token sees.
__device__ __forceinline__ int attention_limit(const AttentionParams& p, const AttentionSeq& s, int token) {
  return p.causal ? max(0, min(s.nk, s.nk - s.nq + token + 1)) : s.nk;
}

}  // namespace vfa
