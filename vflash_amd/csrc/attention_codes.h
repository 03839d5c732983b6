// E4M3 keys and values of a paged cache on their way to the matrix cores.  Kernel-side only; not part of the C-ABI.
#pragma once
#include "attention.h"

namespace vfa {

// Eight E4M3 codes as 16-bit operands of a product; exact.
template <bool F16>
__device__ __forceinline__ v4i attention_widen(v2i c) {
  v4i w;
  static_for<4>([&](auto i) {
    if constexpr (F16)
      w[(int)i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i / 2], 1.0f, (i & 1) != 0));
    else
      w[(int)i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i / 2], 1.0f, (i & 1) != 0));
  });
  return w;
}

// What two bf16 leave of the weights that they were rounded from, as bf16: f16 queries take both, so that their
// results keep f16's precision (16 bits of a weight; binary32's range, which factors need).
__device__ __forceinline__ int attention_rest(float a, float b, int rounded) {
  return pack2<false>(a - bf16_lo((uint32_t)rounded), b - bf16_hi((uint32_t)rounded));
}

}  // namespace vfa
