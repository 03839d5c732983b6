// Rotary positions and the append to a paged cache: the angle of a position, and the place of a token.
#pragma once
#include "common.h"
#include "paged_params.h"

namespace vfa {

// cos and sin of 2 pi phase / 2^32: the octant by integers, then the Taylor series of each on [-pi/4, pi/4]
// (the first terms left out are below 2e-9 and 3e-8 there).
__device__ __forceinline__ v2f cos_sin(uint32_t phase) {
  const uint32_t quadrant = (phase + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(phase - (quadrant << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = x * x;
  float s = __builtin_fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(y, s, 8.3333333e-3f);
  s = __builtin_fmaf(y, s, -1.6666667e-1f);
  s = __builtin_fmaf(x * y, s, x);
  float c = __builtin_fmaf(y, 2.4801587e-5f, -1.3888889e-3f);
  c = __builtin_fmaf(y, c, 4.1666667e-2f);
  c = __builtin_fmaf(y, c, -0.5f);
  c = __builtin_fmaf(y, c, 1.0f);
  const float cc = quadrant & 1 ? s : c, ss = quadrant & 1 ? c : s;
  return v2f{(quadrant + 1) & 2 ? -cc : cc, quadrant & 2 ? -ss : ss};
}

// The sequence of a token: the last whose offset is not past it, by 64 probes at a time.  -1: before the first.
__device__ __forceinline__ int64_t sequence_of(const int64_t* offsets, int64_t batch, int64_t token) {
  int64_t low = 0, count = batch + 1;  // offsets[low .. low + count) hold the answer, or none does
  bool any = false;
  while (count > 0) {
    const int64_t step = (count + 63) / 64, at = step * ((int)threadIdx.x & 63);
    const uint64_t under = __builtin_amdgcn_ballot_w64(at < count && offsets[low + (at < count ? at : 0)] <= token);
    // Offsets that decrease give some sequence or none; every lane of every wave finds the same.
    const int hits = under == ~uint64_t(0) ? 64 : __builtin_ctzll(~under);
    if (hits == 0) return any ? low - 1 : -1;
    any = true;
    const int64_t first = low + step * (hits - 1) + 1;
    const int64_t end = low + (step * hits < count ? step * hits : count);
    low = first;
    count = end - first;
  }
  return low - 1;
}

// Where a token's keys and values go; position -1: nowhere.
struct TokenPlace {
  int64_t position, page;
};
__device__ __forceinline__ TokenPlace token_place(const RotateParams& p, int64_t token) {
  int64_t b = token, after = 1;  // after: the tokens from this one to the sequence's last
  if (p.q_offsets) {
    b = sequence_of(p.q_offsets, p.batch, token);
    if (b < 0 || b >= p.batch) return TokenPlace{-1, 0};
    after = p.q_offsets[b + 1] - token;
  }
  const uint64_t room = (uint64_t)p.cache.width << p.cache.page_shift;
  const uint64_t at = (uint64_t)p.cache.lengths[b] - (uint64_t)after;
  if (at >= room) return TokenPlace{-1, 0};
  const int64_t page = p.cache.table[b * p.cache.width + (int64_t)(at >> p.cache.page_shift)];
  if ((uint64_t)page >= (uint64_t)p.cache.pages) return TokenPlace{-1, 0};
  return TokenPlace{(int64_t)at, page};
}

}  // namespace vfa
