// Rotary positions for gfx950, alone and fused with the append to a paged cache.
//
// A pair (a, b) of a head's values turns by angle position * f:
//   a' = (a cos - b sin) g,  b' = (a sin + b cos) g,   g the magnitude,
// in binary32 with one rounding.  Pair i is (2 i, 2 i + 1) of the head (interleaved) or (i, i + pairs) (half);
// what lies past 2 pairs is copied.
//
// The angle is never a rounded product: f is held as turns, rounded to 2^-64, so that position * f modulo one turn is
// a 64-bit integer product without a rounding of its own, and its upper 32 bits are the phase.  Against the
// frequency itself it is 2^-33 + |position| 2^-65 of a turn off at most: 7e-10 rad, twice that at positions of 2^32,
// 1.9e-7 rad at 2^40.  No table of cosines is read.
//
// Bound by the copy: each value is read and written once.  A workgroup is one wave and takes one token, whose sines and
// cosines it forms once in LDS, a lane a pair, for all heads.  What counts is how many tokens are on their way: 32
// workgroups a CU, by at most 64 registers.  32760 tokens of 80 heads of 128: 265 us, 5.1 TB/s; appending 9200 tokens of 36
// heads, us in waves of 64 registers: one 43, two a workgroup 45, four 51 (and 60 with 67 registers, of which a CU
// holds 28); with four heads a lane loaded ahead (91 registers) 70.
#include "quant_ops.h"
#include "rotary.h"

#include <type_traits>

namespace vfa {

namespace {

constexpr int RT_THREADS = 64;
constexpr int RT_PAIRS = 128;  // at most

// row_divisor for heads that share a wave: fast where all of them are (either way gives the same codes).
__device__ __forceinline__ RowDivisor heads_divisor(float s, float amax) {
  RowDivisor d{s, 1.0f / s, false};
  d.fast = __builtin_amdgcn_ballot_w64(!(amax <= 3.40282347e38f && s >= 0x1p-72f && s <= 3.40282347e38f)) == 0;
  return d;
}

template <bool F16>
__device__ __forceinline__ void widen8(v4i w, float (&x)[8]) {
  if constexpr (F16) {
    const v8hf h = __builtin_bit_cast(v8hf, w);
    static_for<8>([&](auto i) { x[i] = (float)h[(int)i]; });
  } else {
    static_for<4>([&](auto i) {
      x[2 * i] = bf16_lo((uint32_t)w[(int)i]);
      x[2 * i + 1] = bf16_hi((uint32_t)w[(int)i]);
    });
  }
}
template <bool F16>
__device__ __forceinline__ float widen1(uint16_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, w);
  else return bf16_to_f32(w);
}
template <bool F16>
__device__ __forceinline__ v4i narrow8(const float (&x)[8]) {
  v4i w;
  static_for<4>([&](auto i) {
    if constexpr (F16) w[(int)i] = __builtin_bit_cast(int, v2hf{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
    else w[(int)i] = (int)pack_bf16x2(x[2 * i], x[2 * i + 1]);
  });
  return w;
}

}  // namespace

// One token, the heads of blockIdx.z: 2^lanes_shift lanes a head, eight d a lane.  Heads [0, heads) are q's,
// [heads, heads + key_heads) k's and, with a cache, as many of v's.
template <bool F16>
__global__ void __launch_bounds__(RT_THREADS, 8) rotate_heads(const RotateParams p, int lanes_shift, int heads_per_group) {
  __shared__ float cosines[RT_PAIRS], sines[RT_PAIRS];
  const int64_t token = grid_row();
  if (token >= p.tokens) return;
  const RotaryParams& r = p.rotary;
  const bool cached = p.cache.values != nullptr;

  const TokenPlace place = cached ? token_place(p, token) : TokenPlace{-1, 0};
  const int64_t position = place.position, page = place.page;
  if (r.phases) {
    for (int i = (int)threadIdx.x; i < r.pairs; i += RT_THREADS) {
      const int64_t axis = r.axis ? r.axis[i] : 0;
      const int64_t at = !r.positions ? position : (uint64_t)axis < (uint64_t)r.axes ? r.positions[token * r.axes + axis] : 0;
      const uint64_t turn = (uint64_t)at * r.phases[i];
      const v2f cs = cos_sin((uint32_t)((turn + 0x80000000ull) >> 32));
      cosines[i] = cs[0] * r.magnitude;
      sines[i] = cs[1] * r.magnitude;
    }
    __syncthreads();
  }

  const int lanes = 1 << lanes_shift, d = 8 * ((int)threadIdx.x & (lanes - 1));
  const int all = (p.q_out ? p.heads : 0) + (cached ? 2 : 1) * p.key_heads;
  const int first = p.q_out ? 0 : p.heads;  // heads of q that are left out
  const int end = min((int)(blockIdx.z + 1) * heads_per_group, all);
  for (int h = blockIdx.z * heads_per_group + ((int)threadIdx.x >> lanes_shift); h < end; h += RT_THREADS >> lanes_shift) {
    const int head = h + first;
    const bool is_q = head < p.heads, is_v = head >= p.heads + p.key_heads;
    const int g = is_q ? head : head - p.heads - (is_v ? p.key_heads : 0);
    const uint16_t* src = is_q ? p.q + token * p.q_ts + g * p.q_hs
                          : is_v ? p.v + token * p.v_ts + g * p.v_hs : p.k + token * p.k_ts + g * p.k_hs;
    const bool live = d < p.dim;
    float x[8] = {};
    if (live) {
      widen8<F16>(*reinterpret_cast<const v4i*>(src + d), x);
      if (r.phases && !is_v && d < 2 * r.pairs) {
        if (r.interleaved) {
          static_for<4>([&](auto i) {
            const int pair = d / 2 + i;
            if (pair < r.pairs) {
              const float c = cosines[pair], s = sines[pair], a = x[2 * i], b = x[2 * i + 1];
              x[2 * i] = a * c - b * s;
              x[2 * i + 1] = a * s + b * c;
            }
          });
        } else {
          float other[8];
          const int shift = r.pairs;
          if (r.pairs % 8 == 0) {
            widen8<F16>(*reinterpret_cast<const v4i*>(src + (d < shift ? d + shift : d - shift)), other);
          } else {
            static_for<8>([&](auto i) {
              const int e = d + i;
              other[i] = e < 2 * shift ? widen1<F16>(src[e < shift ? e + shift : e - shift]) : 0.0f;
            });
          }
          static_for<8>([&](auto i) {
            const int e = d + i;
            if (e < 2 * shift) {
              const int pair = e < shift ? e : e - shift;
              const float s = sines[pair];
              x[i] = x[i] * cosines[pair] + other[i] * (e < shift ? -s : s);
            }
          });
        }
      }
    }
    if (is_q || !cached) {
      uint16_t* dst = is_q ? p.q_out + (token * p.heads + g) * p.dim : p.k_out + (token * p.key_heads + g) * p.dim;
      if (live) *reinterpret_cast<v4i*>(dst + d) = cached && position < 0 ? v4i{} : narrow8<F16>(x);
      continue;
    }
    const int64_t slot = (((page * 2 + (is_v ? 1 : 0)) * p.key_heads + g) << p.cache.page_shift) +
                         (position & ((int64_t(1) << p.cache.page_shift) - 1));
    if (!p.cache.scales) {
      if (live && position >= 0) *reinterpret_cast<v4i*>(p.cache.values + 2 * (slot * p.dim + d)) = narrow8<F16>(x);
      continue;
    }
    // E4M3: the scale and the quotients of the row quantizer, from the unrounded values.
    float top = 0;
    static_for<8>([&](auto j) { top = nan_max(top, fabsf(x[j])); });
    for (int o = 1; o < lanes; o <<= 1) top = nan_max(top, __shfl_xor(top, o, 64));
    const RowDivisor by = heads_divisor(row_scale(top), top);
    uint2 codes;
    if (by.fast) {
      float q[8];
      static_for<8>([&](auto j) { q[j] = clamped_row_quotient<true>(x[j], by); });
      codes.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false), true);
      codes.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false), true);
    } else {
      uint32_t code[8];
      static_for<8>([&](auto j) { code[j] = quant1(x[j], by.s); });
      codes = make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
    }
    if (position < 0) continue;
    if (live) *reinterpret_cast<uint2*>(p.cache.values + slot * p.dim + d) = codes;
    if (d == 0) p.cache.scales[slot] = by.s;
  }
}

int compute_units();

hipError_t launch_rotate(const RotateParams& p, hipStream_t s) {
  int lanes_shift = 0;
  while ((8 << lanes_shift) < p.dim) ++lanes_shift;
  const int all = (p.q_out ? p.heads : 0) + (p.cache.values ? 2 : 1) * p.key_heads;
  // Few tokens are spread over more workgroups, up to twice what the GPU holds.
  const int rows = RT_THREADS >> lanes_shift, times = (all + rows - 1) / rows;  // heads at a time
  int64_t parts = 64 * (int64_t)compute_units() / p.tokens;
  if (parts > 1024) parts = 1024;
  parts = parts < 1 ? 1 : parts > times ? times : parts;
  const int per = (times + (int)parts - 1) / (int)parts * rows;
  dim3 grid = row_grid(p.tokens);
  grid.z = (unsigned)((all + per - 1) / per);
  if (p.f16) rotate_heads<true><<<grid, RT_THREADS, 0, s>>>(p, lanes_shift, per);
  else rotate_heads<false><<<grid, RT_THREADS, 0, s>>>(p, lanes_shift, per);
  return hipGetLastError();
}

}  // namespace vfa
