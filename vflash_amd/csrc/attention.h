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

typedef short v4s16 __attribute__((ext_vector_type(4)));

// Below every finite exponent: 2^(x - m) is 0 for a masked x = -inf, with no inf - inf.
#define VFA_LOWEST (-3.4028234663852886e38f)
// A weight carries 2^shift, and m follows the scores only where a block's weights would sum up to more
// than a bound above that.  A rounding is relative, so a weight above that of m loses nothing.
// bf16: 2^20 above, and a shift by which all keys at the bound sum up to 2^-1: no sum of finite values
// overflows before it is normalised (values below 2^(-126 - shift) enter it as subnormals).  A bound of
// 2^9 instead costs 5 % where the scores spread by 10 and 8 % where they rise by 0.05 a key (6000
// tokens, 16 heads of 128: 300 and 306 us).  f16: 2^6 keeps 20 binary orders below m out of the weights'
// subnormals, and 2^15 them from overflowing.  Tiles of few rows, which wait for their keys, follow the
// maximum itself, once it is 2^8 above.
template <bool F16>
__device__ __forceinline__ float attention_shift(const AttentionParams& p) { return F16 ? 6.0f : p.shift; }
template <bool F16>
__device__ __forceinline__ float attention_bound(const AttentionParams& p) { return F16 ? 32768.0f : p.bound; }
constexpr float kAttentionSlack = 8.0f;
constexpr float kAttentionFar = 4194304.0f;  // 2^22: a rounding of 1/4

// 2^(c (s - m)) times 2^shift, m the row's maximum before its scaling (ref = shift - c m).
template <bool FAR>
__device__ __forceinline__ float attention_weight(float s, float c, float m, float ref, float shift) {
  return __builtin_amdgcn_exp2f(FAR ? (s - m) * c + shift : __builtin_fmaf(s, c, ref));
}
// l plus the two weights of a packed pair, as they were rounded: the sum that normalises them
// over values in the operands' type, so that what their roundings have in common cancels (a value that
// all keys share comes back as it is).  Over E4M3 pages a weight is rounded with its value's factor, and the
// sum is that of the unrounded weights: errors against 64 bits are 1.4 times those of weights in 32 bits.
template <bool F16>
__device__ __forceinline__ float attention_sum2(int pair, float l) {
  if constexpr (F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2hf, pair), v2hf{(_Float16)1.0f, (_Float16)1.0f}, l, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), v2bf{(__bf16)1.0f, (__bf16)1.0f}, l, false);
}
// A row's maximum as its statistics carry it: scaled, and finite where it saw nothing.
__device__ __forceinline__ float attention_top(float m, float c) { return fmaxf(m * c, VFA_LOWEST); }

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

// Inclusive prefix maximum of values that are not negative.
__device__ __forceinline__ int wave_scan_max(int v, int lane) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true));
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31);
  const int r2 = __builtin_amdgcn_readlane(v, 47);
  return max(v, lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? max(r0, r1) : max(r0, max(r1, r2)));
}

struct AttentionSeq {
  int q0, k0, nq, nk;
};
// This lane's sequence, base + lane of 0 .. batch + 1 (0 and batch + 1: the rows outside the
// offsets).  Sequences begin where the one before ends, at the running maximum of the offsets, so
// that they cover every row once whatever these hold; `reached` carries it from base to base.
// With PAGED, k0 is the sequence itself, 0 .. batch - 1.
template <bool PAGED = false>
__device__ __forceinline__ AttentionSeq attention_sequence(const AttentionParams& p, int64_t base, int& reached) {
  // Clamped to [0, hi] through the 32 bits that are left when the others say which side.
  auto clamp = [](int64_t v, int hi) { return v < 0 ? 0 : (uint64_t)v > (uint64_t)hi ? hi : (int)v; };
  const int64_t s = base + (threadIdx.x & 63);
  const bool real = s > 0 && s <= p.batch;
  // Every lane loads, from a place that exists, so that no load waits for another.
  const int64_t at = s < 1 ? 0 : s > p.batch ? p.batch : s, before = at > 0 ? at - 1 : 0;
  int64_t from = before, to = at;  // a token a sequence
  if (!PAGED || p.q_offsets) {
    from = p.q_offsets[before];
    to = p.q_offsets[at];
  }
  int64_t k0 = 0, kn = 0;
  if (p.batch) {
    if constexpr (PAGED) {
      kn = p.cache.lengths[before];
    } else {
      k0 = p.k_offsets[before];
      kn = (p.k_lengths ? p.k_lengths : p.k_offsets + 1)[before];
    }
  }
  // Sequence batch + 1 begins where the offsets end; later ones are empty.
  const int first = s == 0 ? 0 : clamp(s > p.batch ? to : from, p.tokens);
  AttentionSeq r;
  r.q0 = max(reached, wave_scan_max(first, (int)threadIdx.x & 63));
  r.nq = s > p.batch + 1 ? 0 : max(0, (s > p.batch ? p.tokens : clamp(to, p.tokens)) - r.q0);
  if constexpr (PAGED) {
    r.k0 = (int)before;
    r.nk = real ? clamp(kn, p.keys) : 0;
  } else {
    r.k0 = clamp(k0, p.keys);
    r.nk = !real ? 0 : p.k_lengths ? clamp(kn, p.keys - r.k0) : max(0, clamp(kn, p.keys) - r.k0);
  }
  reached = __builtin_amdgcn_readlane(r.q0 + r.nq, 63);
  return r;
}

__device__ __forceinline__ uint32_t attention_tiles_of(const AttentionParams& p, const AttentionSeq& s) {
  return (uint32_t)(((uint64_t)((uint32_t)s.nq + (uint32_t)p.tile_tokens - 1) * p.tile_mul) >> p.tile_shift);
}

struct AttentionItem {
  AttentionSeq seq;  // all uniform
  int tile;          // of the sequence
  int split, splits;
  int chunk;         // keys of a split
  int slot;          // of the tile's split 0, where it has several
  int head_block;
  bool live;
};

// a / b of values that a wave shares; most are small enough to go without the division.
__device__ __forceinline__ uint32_t attention_quotient(uint32_t a, uint32_t b) {
  return a < b ? 0 : a < 2 * b ? 1 : b == 1 ? a : a / b;
}
// The key head of a head block, and which of its parts this is.
__device__ __forceinline__ int attention_key_head(const AttentionParams& p, int head_block) {
  return p.parts == 1 ? head_block : head_block / p.parts;
}

// Which of `total` units of which head block workgroup `index` takes; false: none.
// Workgroup b runs on XCD b % 8.  Where the head blocks divide among the XCDs, each XCD takes whole
// ones, one after another, so that its L2 holds their keys.  Causal tiles differ in length: a
// head goes from its longest to its shortest and the next one back, so that the tiles that meet on
// a CU are long and short, and the last ones are short.
__device__ __forceinline__ bool attention_place(const AttentionParams& p, uint32_t index, int total, int& head_block, int& x) {
  if (total == 0) return false;
  if (p.head_blocks % 8 == 0) {
    const int i = (int)(index >> 3), each = p.head_blocks / 8;
    const int local = (int)attention_quotient((uint32_t)i, (uint32_t)total);
    if (local >= each) return false;
    head_block = (int)(index & 7) + 8 * local;
    x = i - local * total;
    if (p.causal && (each - 1 - local) % 2) x = total - 1 - x;
    return true;
  }
  x = (int)attention_quotient(index, (uint32_t)p.head_blocks);
  head_block = (int)index - x * p.head_blocks;
  return x < total;
}

// The unit `index` of the launch: an item, or with JOIN a tile (all its splits).
template <bool JOIN, bool PAGED = false>
__device__ __forceinline__ AttentionItem attention_find(const AttentionParams& p, uint32_t index) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t n = p.batch + 2;
  int reached = 0, x;
  AttentionItem it{};
  AttentionSeq mine = attention_sequence<PAGED>(p, 0, reached);
  auto take = [&](int l) {
    auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
    it.seq = AttentionSeq{pick(mine.q0), pick(mine.k0), pick(mine.nq), pick(mine.nk)};
    it.live = true;
  };
  if (!p.target && n <= 64) {  // no split, and the sequences are in the lanes
    const int t = (int)attention_tiles_of(p, mine);
    int total;
    const int incl = wave_scan(t, lane, total);
    if (!attention_place(p, index, total, it.head_block, x)) return it;
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > x));
    take(l);
    it.tile = __builtin_amdgcn_readlane(incl, l) - 1 - x;  // from the last to the first: longest first
    it.splits = 1;
    it.chunk = INT32_MAX;
    return it;
  }
  auto blocks_of = [](const AttentionSeq& s) { return ((uint32_t)s.nk + 63) >> 6; };
  // Keys of a split, in blocks of 64: the whole sequence where the tiles fill the GPU, else as
  // many as make about p.target items.
  uint32_t chunk = 1u << 25;
  int tiles = 0;
  auto each = [&](auto&& f) {  // f(tiles) for every 64 sequences, in `mine`, until it returns true
    reached = 0;
    for (int64_t base = 0; base < n; base += 64) {
      if (n > 64) mine = attention_sequence<PAGED>(p, base, reached);
      if (f((int)attention_tiles_of(p, mine))) return;
    }
  };
  if (p.target) {
    float work = 0;
    each([&](int t) {
      int sum;
      wave_scan(t, lane, sum);
      tiles += sum;
      work += wave_sum((float)t * (float)blocks_of(mine));
      return false;
    });
    work = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(work)));
    chunk = max((uint32_t)p.min_chunk, (uint32_t)fminf(ceilf(work * (float)p.head_blocks / (float)p.target), 33554432.0f));
  }
  auto splits_of = [&](const AttentionSeq& s) { return (int)max(1u, (blocks_of(s) + chunk - 1) / chunk); };
  auto slots_of = [](int t, int sp) { return sp > 1 ? t * sp : 0; };
  // Units and slots per head block; the grid's order needs them before the search.  A split
  // sequence has more keys than a chunk, so the slots are at most 2 p.target.
  int units = 0, slots = 0;
  each([&](int t) {
    const int sp = splits_of(mine);
    int sum;
    wave_scan(t * sp, lane, sum);
    units += sum;
    wave_scan(slots_of(t, sp), lane, sum);
    slots += sum;
    return false;
  });
  if (p.target && (int64_t)slots * p.head_blocks > p.slots) {  // not reached: a bound on the memory
    chunk = 1u << 25;
    units = tiles;
  }
  if (!attention_place(p, index, JOIN ? tiles : units, it.head_block, x)) return it;
  int before = 0, slots_before = 0;
  each([&](int t) {
    const int sp = splits_of(mine), own = JOIN ? t : t * sp;
    int sum, slot_sum;
    const int incl = wave_scan(own, lane, sum);
    const int slot_incl = wave_scan(slots_of(t, sp), lane, slot_sum);
    if (x < before + sum) {
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + incl > x));
      take(l);
      it.splits = __builtin_amdgcn_readlane(sp, l);
      const int in = x - before - __builtin_amdgcn_readlane(incl - own, l);
      const int back = JOIN ? in : in / it.splits;
      it.split = JOIN ? 0 : in - back * it.splits;
      it.tile = __builtin_amdgcn_readlane(t, l) - 1 - back;
      it.chunk = (int)min((uint64_t)chunk * 64, (uint64_t)INT32_MAX);
      it.slot = it.head_block * slots + slots_before + __builtin_amdgcn_readlane(slot_incl - slots_of(t, sp), l) +
                back * it.splits;
      return true;
    }
    before += sum;
    slots_before += slot_sum;
    return false;
  });
  return it;
}

// The same in scalar registers, where the compiler does not see that the search is uniform.
template <bool JOIN, bool PAGED = false>
__device__ __forceinline__ AttentionItem attention_item(const AttentionParams& p, uint32_t index) {
  auto u = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const AttentionItem f = attention_find<JOIN, PAGED>(p, index);
  AttentionItem it;
  it.seq = AttentionSeq{u(f.seq.q0), u(f.seq.k0), u(f.seq.nq), u(f.seq.nk)};
  it.tile = u(f.tile);
  it.split = u(f.split);
  it.splits = u(f.splits);
  it.chunk = u(f.chunk);
  it.slot = u(f.slot);
  it.head_block = u(f.head_block);
  it.live = u(f.live) != 0;
  return it;
}

// Row r of a tile: its token in the sequence, its head, and whether it is one.
struct AttentionRow {
  int token, head;
  bool live;
};
// Row r's token of the tile: r / heads_per_tile, for r < 512.
__device__ __forceinline__ int attention_token_of(const AttentionParams& p, int r) { return (r * p.row_mul) >> 16; }
__device__ __forceinline__ AttentionRow attention_row(const AttentionParams& p, const AttentionItem& it, int r) {
  const int in = attention_token_of(p, r);
  const int key_head = attention_key_head(p, it.head_block);
  const int h = (it.head_block - key_head * p.parts) * p.heads_per_tile + r - in * p.heads_per_tile;
  AttentionRow row;
  row.token = it.tile * p.tile_tokens + in;
  row.head = key_head * p.group + h;
  row.live = in < p.tile_tokens && row.token < it.seq.nq && h < p.group;
  return row;
}

// Eight d of the row, zeros past the head's dimension and for a row that is none.  Always a load, from
// a place that exists.
__device__ __forceinline__ v4i attention_query(const AttentionParams& p, const AttentionItem& it, const AttentionRow& row, int d) {
  const uint16_t* src = row.live ? p.q + (int64_t)(it.seq.q0 + row.token) * p.q_ts + (int64_t)row.head * p.q_hs : p.q;
  const v4i v = *reinterpret_cast<const v4i*>(src + min(d, p.dim - 8));
  return row.live && d < p.dim ? v : v4i{};
}

// Keys that the token sees.
__device__ __forceinline__ int attention_limit(const AttentionParams& p, const AttentionSeq& s, int token) {
  return p.causal ? max(0, min(s.nk, s.nk - s.nq + token + 1)) : s.nk;
}

// The schedule of attention_step.  Every tile is a number of units (2^p.unit_shift keys each, one at
// least), the units of all tiles of a head block form a line, the head blocks' lines one after
// another a longer one, and each workgroup takes the next p.grid-th part of that: equal work whatever
// the lengths, where the plan splits keys (else a unit is a whole sequence).  A workgroup whose part ends inside a tile leaves a partial sum, of which it has at
// most two: one of a tile begun by an earlier workgroup (slot 2 b), one of a tile that a later one ends
// (slot 2 b + 1).  On one XCD's workgroups lie whole head blocks where these divide among the XCDs.
struct AttentionLine {
  uint32_t units;       // per head block
  uint32_t quota, end;  // of a workgroup; of the line
  int unit_shift;
  int xcds;             // 8: the line is one XCD's
  AttentionSeq mine;    // of this lane, where there are at most 64 sequences
  // Over a paged cache, one token a sequence: this lane's run of `run` sequences and the lanes' before it, in units.
  int64_t run;
  uint32_t own, upto;
};
struct AttentionSegment {
  AttentionItem it;  // seq, tile, head_block
  uint32_t first, count, of;  // units: the segment's first in its tile, its own, the tile's
};

__device__ __forceinline__ uint32_t attention_units_of(const AttentionLine& l, const AttentionSeq& s) {
  return max(1u, ((uint32_t)s.nk + (1u << l.unit_shift) - 1) >> l.unit_shift);
}

// Over a paged cache, one token a sequence: a sequence is a tile, and the workgroup that ends one goes on with the next.
__device__ __forceinline__ int attention_keys(const AttentionParams& p, int64_t length) {
  return length < 0 ? 0 : length < p.keys ? (int)length : p.keys;
}
// A sequence that the wave shares, by a scalar load.
__device__ __forceinline__ AttentionSeq attention_single(const AttentionParams& p, int64_t sequence) {
  typedef const __attribute__((address_space(4))) int64_t lengths_t;
  const int s = __builtin_amdgcn_readfirstlane((int)sequence);
  return AttentionSeq{s, s, 1, attention_keys(p, ((lengths_t*)(uintptr_t)p.cache.lengths)[s])};
}
// Of whole sequences, unit i of a head block is sequence i.
__device__ __forceinline__ bool attention_direct(const AttentionParams& p) { return !p.q_offsets && p.unit_shift == 31; }

template <bool PAGED = false>
__device__ __forceinline__ AttentionLine attention_line(const AttentionParams& p, int grid) {
  const int lane = (int)threadIdx.x & 63;
  AttentionLine l{};
  l.unit_shift = p.unit_shift;
  int reached = 0;
  const bool singles = PAGED && !p.q_offsets;
  if (PAGED && attention_direct(p)) {
    l.units = (uint32_t)p.batch;
  } else if (singles) {
    // A lane's loads do not wait for each other, and one scan serves any number of sequences.
    l.run = (p.batch + 63) / 64;
    const int64_t s0 = lane * l.run, s1 = s0 + l.run < p.batch ? s0 + l.run : p.batch;
#pragma unroll 4
    for (int64_t s = s0; s < s1; ++s) l.own += attention_units_of(l, AttentionSeq{0, 0, 1, attention_keys(p, p.cache.lengths[s])});
    int sum;
    l.upto = (uint32_t)wave_scan((int)l.own, lane, sum);
    l.units = (uint32_t)sum;
  }
  for (int64_t base = 0; base < p.batch + 2 && !singles; base += 64) {
    l.mine = attention_sequence<PAGED>(p, base, reached);
    int sum;
    wave_scan((int)(attention_tiles_of(p, l.mine) * attention_units_of(l, l.mine)), lane, sum);
    l.units += (uint32_t)sum;
  }
  l.xcds = p.head_blocks % 8 == 0 ? 8 : 1;
  const int shift = l.xcds == 8 ? 3 : 0;
  l.end = l.units * (uint32_t)(p.head_blocks >> shift);
  const uint32_t parts = (uint32_t)grid >> shift;
  l.quota = max(PAGED ? p.least_units : 1u, attention_quotient(l.end + parts - 1, parts));
  return l;
}

// The rest of the tile at unit `pos` (< line.end) of workgroup b's line, up to unit `stop`.
template <bool PAGED = false>
__device__ __forceinline__ AttentionSegment attention_segment(const AttentionParams& p, const AttentionLine& line, int b,
                                                              uint32_t pos, uint32_t stop) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t n = p.batch + 2;
  AttentionSegment g{};
  const uint32_t local = attention_quotient(pos, line.units), x = pos - local * line.units;
  g.it.head_block = line.xcds == 8 ? (b & 7) + 8 * (int)local : (int)local;
  if (PAGED && !p.q_offsets) {
    auto take = [&](int64_t s, uint32_t before) {
      g.it.seq = attention_single(p, s);
      g.of = attention_units_of(line, g.it.seq);
      g.first = x - before;
      g.count = min(g.of - g.first, stop - pos);
      g.it.live = true;
    };
    if (attention_direct(p)) {
      take(x, x);
      return g;
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(line.upto > x));
    const int64_t s0 = l * line.run, s1 = s0 + line.run < p.batch ? s0 + line.run : p.batch;
    uint32_t before = (uint32_t)__builtin_amdgcn_readlane((int)(line.upto - line.own), l);
    for (int64_t base = s0; base < s1; base += 64) {
      const int64_t s = base + lane;
      const int own = s < s1 ? (int)attention_units_of(line, AttentionSeq{0, 0, 1, attention_keys(p, p.cache.lengths[s])}) : 0;
      int sum;
      const uint32_t incl = (uint32_t)wave_scan(own, lane, sum);
      if (x < before + (uint32_t)sum) {
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + incl > x));
        take(base + at, before + (uint32_t)__builtin_amdgcn_readlane((int)incl - own, at));
        return g;
      }
      before += (uint32_t)sum;
    }
    return g;
  }
  uint32_t before = 0;
  int reached = 0;
  for (int64_t base = 0; base < n; base += 64) {
    const AttentionSeq mine = n > 64 ? attention_sequence<PAGED>(p, base, reached) : line.mine;
    const uint32_t u = attention_units_of(line, mine), own = attention_tiles_of(p, mine) * u;
    int sum;
    const uint32_t incl = (uint32_t)wave_scan((int)own, lane, sum);
    if (x < before + (uint32_t)sum) {
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + incl > x));
      auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      g.it.seq = AttentionSeq{pick(mine.q0), pick(mine.k0), pick(mine.nq), pick(mine.nk)};
      g.of = (uint32_t)pick((int)u);
      const uint32_t in = x - before - (uint32_t)pick((int)(incl - own));
      g.it.tile = (int)attention_quotient(in, g.of);
      g.first = in - (uint32_t)g.it.tile * g.of;
      g.count = min(g.of - g.first, stop - pos);
      g.it.live = true;
      return g;
    }
    before += (uint32_t)sum;
  }
  return g;
}

// The segment at `pos`, behind one that ends its tile there.
template <bool PAGED>
__device__ __forceinline__ AttentionSegment attention_following(const AttentionParams& p, const AttentionLine& line, int b,
                                                                const AttentionSegment& ended, uint32_t pos, uint32_t stop) {
  if (!PAGED || p.q_offsets) return attention_segment<PAGED>(p, line, b, pos, stop);
  AttentionSegment g = ended;
  int s = ended.it.seq.k0 + 1;
  if (s == p.batch) {
    s = 0;
    g.it.head_block += line.xcds;
  }
  g.it.seq = attention_single(p, s);
  g.of = attention_units_of(line, g.it.seq);
  g.first = 0;
  g.count = min(g.of, stop - pos);
  return g;
}

// The tile that a workgroup of attention_step began and others end: its segments (0: none), its first row of
// q, its tokens and its head block.  Over a paged cache it is left in memory for the join, which finds it again from
// the lengths otherwise: 15 sequences of four tokens 21.2 us, 23.8 without; one of 8000 keys, four tokens 24.2 and 25.4.
struct AttentionBegun {
  int segments, row, tokens, head_block;
};
// `seg`: the last that the workgroup took, up to `stop`.
__device__ __forceinline__ AttentionBegun attention_begun(const AttentionParams& p, const AttentionLine& line, int b,
                                                          const AttentionSegment& seg, uint32_t stop) {
  if (!seg.it.live || seg.first || seg.count == seg.of) return AttentionBegun{};
  const int segments = (int)((stop - seg.count + seg.of - 1) / line.quota) - (b >> (line.xcds == 8 ? 3 : 0)) + 1;
  const int row = seg.it.tile * p.tile_tokens;
  return AttentionBegun{segments, seg.it.seq.q0 + row, min(p.tile_tokens, seg.it.seq.nq - row), seg.it.head_block};
}

// In scalar registers, where the compiler does not see that the search is uniform.
__device__ __forceinline__ AttentionSegment attention_scalar(const AttentionSegment& g) {
  auto u = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  AttentionSegment s{};
  s.it.seq = AttentionSeq{u(g.it.seq.q0), u(g.it.seq.k0), u(g.it.seq.nq), u(g.it.seq.nk)};
  s.it.tile = u(g.it.tile);
  s.it.head_block = u(g.it.head_block);
  s.it.live = u(g.it.live) != 0;
  s.first = (uint32_t)u((int)g.first);
  s.count = (uint32_t)u((int)g.count);
  s.of = (uint32_t)u((int)g.of);
  return s;
}

}  // namespace vfa
