// NVFP4-weight linear with 16-bit activations (weight-only) for gfx950.
//
//   out[m, n] = bf16(alpha * sum_k x[m, k] * e2m1(w[n, k]) * e4m3(s[n, k / 16]) + bias[n])
//
// x is bf16 or f16 and enters as it is.  A product e2m1 * e4m3 has at most 6 significant bits and
// lies in 2^-10 .. 2688, so it is exact in bf16 and in f16: the only roundings are those of the
// binary32 sum and the last one.  Scales in the 128x4 order of nvfp4_gemm.hip.
//
// Two kernels, chosen by the sizes (launch_nvfp4_w16):
//   nvfp4_w16_few   up to 64 rows a workgroup, bound by the weight's bytes;
//   nvfp4_w16_pipe  tiles of many rows, bound by the MFMAs and the conversions that feed them.
// Both restore the weight in registers: eight values cost 8 VALU instructions in f16 (the packed
// multiply takes the scale) and 16 in bf16, which has none (conversion to binary32, multiply,
// rounding, exact all the same).
#include "gemm_epilogue.h"

#include <type_traits>

namespace vfa {

typedef _Float16 w16_v2h __attribute__((ext_vector_type(2)));
typedef _Float16 w16_v8h __attribute__((ext_vector_type(8)));

// A lane's scales: two neighbouring E4M3 block scales in the low half of `bytes`.
template <bool F16>
struct W16Scales {
  v2f f;
  w16_v2h h;
  __device__ __forceinline__ explicit W16Scales(uint32_t bytes) {
    if constexpr (F16) h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 1.0f, false);
    else f = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes, false);
  }
};

// The eight values of packed word d times block scale I of s, as an MFMA operand.
template <bool F16, int I>
__device__ __forceinline__ v4i w16_restore(uint32_t d, const W16Scales<F16>& s) {
  v4i o;
  static_for<4>([&](auto i) {
    if constexpr (F16) {
      o[(int)i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, 1.0f, (int)i) * w16_v2h{s.h[I], s.h[I]});
    } else {
      const v2f y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, (int)i);
      const float a = y[0] * s.f[I], b = y[1] * s.f[I];
      o[(int)i] = (int)pack_bf16x2(a, b);
    }
  });
  return o;
}

template <bool F16>
__device__ __forceinline__ v16f w16_mfma32(v4i a, v4i b, v16f c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(w16_v8h, a), __builtin_bit_cast(w16_v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ v4f w16_mfma16(v4i a, v4i b, v4f c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(w16_v8h, a), __builtin_bit_cast(w16_v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Few rows.  A workgroup computes 16 MB rows of x times 16 NB rows of the weight, and its eight
// waves take every eighth piece of 128 K, loaded straight into registers D pieces ahead: lane
// (i, g) of a piece holds 32 K of weight row i (16 bytes), the two scales they need and the
// matching K of the x rows, in the order that makes them four MFMA steps of 8 K a lane.  The
// waves' sums meet in LDS.  The 16-row blocks of a workgroup lie 32 rows apart, as the scales of
// one 16-byte run do.
template <bool F16, int NB, int MB, int D>
__global__ void __launch_bounds__(512, 2) nvfp4_w16_few(const GemmParams p, int blocks_m) {
  constexpr int WAVES = 8, SUBS = 8 / NB, PITCH = 16 * NB + 4;
  __shared__ float sums[WAVES][16 * MB * PITCH];
  // A 128-row tile's workgroups run on one XCD, whose L2 then serves the scales and weights that
  // they share.
  const int per_tile = SUBS * blocks_m;
  const int xcd = (int)blockIdx.x & 7, j = (int)blockIdx.x >> 3;
  const int64_t tile = (int64_t)(j / per_tile) * 8 + xcd;
  if (tile >= p.n / 128) return;
  const int sub = j % per_tile % SUBS;
  const int64_t m0 = (int64_t)(j % per_tile / SUBS) * (16 * MB);
  const int half = sub & 1, b0 = (sub >> 1) * NB;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = (int)threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int64_t k_tiles = p.k / 64;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + tile * 128 * p.ldw, (uint32_t)(128 * p.ldw));
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.wsb + tile * k_tiles * 512, (uint32_t)(k_tiles * 512));
  const int64_t rows = min((int64_t)(16 * MB), p.m - m0);
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.a + m0 * p.lda, (uint32_t)(rows * p.lda));
  const uint32_t w_row = (uint32_t)((32 * b0 + 16 * half + i) * p.ldw);
  const uint32_t s_row = (uint32_t)((16 * half + i) * 16 + b0 * 4);
  struct Piece {
    v4i w[NB];
    uint32_t s[NB];
    v4i x[MB][4];
  };
  auto load = [&](Piece& q, int64_t c) {
    const int64_t k = 128 * c + 32 * g;
    const bool live = k < p.k;
    static_for<NB>([&](auto b) {
      q.w[b] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
                                           rw, live ? w_row + (uint32_t)(b * 32 * p.ldw + k / 2) : VFA_OOB, 0, 0));
    });
    const uint32_t so = live ? s_row + (uint32_t)(k / 64 * 512) : VFA_OOB;
    if constexpr (NB == 4) {
      const v4i s = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rs, so, 0, 0));
      static_for<4>([&](auto b) { q.s[b] = (uint32_t)s[(int)b]; });
    } else {
      static_for<NB>([&](auto b) { q.s[b] = __builtin_amdgcn_raw_buffer_load_b32(rs, so + 4 * b, 0, 0); });
    }
    static_for<MB>([&](auto m) {
      static_for<4>([&](auto v) {
        q.x[m][v] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
                                                rx, live ? (uint32_t)((16 * m + i) * p.lda + 2 * k + 16 * v) : VFA_OOB, 0, 0));
      });
    });
  };
  v4f acc[NB][MB];
  static_for<NB>([&](auto b) { static_for<MB>([&](auto m) { acc[b][m] = v4f{}; }); });
  auto multiply = [&](const Piece& q) {
    static_for<NB>([&](auto b) {
      const W16Scales<F16> s(q.s[b] >> (16 * (g & 1)));
      static_for<4>([&](auto v) {
        const v4i w = w16_restore<F16, v / 2>((uint32_t)q.w[b][(int)v], s);
        static_for<MB>([&](auto m) { acc[b][m] = w16_mfma16<F16>(w, q.x[m][v], acc[b][m]); });
      });
    });
  };
  const int64_t pieces = (p.k + 127) / 128;
  Piece q[D];
  static_for<D>([&](auto d) { load(q[d], wave + WAVES * d); });
  for (int64_t c = wave; c < pieces; c += WAVES * D)
    static_for<D>([&](auto d) {
      multiply(q[d]);  // zeros past the last piece
      load(q[d], c + WAVES * (D + d));
    });
  // Lane (m, g) holds the weight rows 4 g .. + 3 of its blocks.
  static_for<NB>([&](auto b) {
    static_for<MB>([&](auto m) {
      *reinterpret_cast<v4f*>(&sums[wave][(16 * m + i) * PITCH + 16 * b + 4 * g]) = acc[b][m];
    });
  });
  __syncthreads();
  const float alpha = *p.sw;
  for (int e = (int)threadIdx.x; e < 16 * MB * 4 * NB; e += 64 * WAVES) {
    const int m = e / (4 * NB), c = e % (4 * NB) * 4;
    if (m >= rows) break;
    v4f y = v4f{};
    static_for<WAVES>([&](auto w) { y += *reinterpret_cast<const v4f*>(&sums[w][m * PITCH + c]); });
    const int64_t n = tile * 128 + 32 * (b0 + c / 16) + 16 * half + c % 16;
    uint32_t o[4];
    static_for<4>([&](auto r) {
      const float z = y[(int)r] * alpha;
      o[r] = f32_to_bf16(p.bias ? z + bf16_to_f32(p.bias[n + r]) : z);
    });
    *reinterpret_cast<uint2*>(p.out + (m0 + m) * p.ldo + n) = make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
  }
}

// ---------------------------------------------------------------------------
// Many rows.  A stage holds 64 K of the tile (activation rows of 128 bytes, packed rows of 32,
// 512 bytes of scales per 128 weight rows) in an LDS ring that DMA fills NS - 1 stages ahead,
// with one barrier a stage.  K goes to the lanes as in w8a16_gemm.hip: a lane reads 64 bytes of an
// activation row and 16 of a packed row.  Four waves lie side by side along N where the tile is
// wide, so that none restores another's weights, and two workgroups share a CU: the MFMAs of one
// run under the conversions and the waits of the other.
template <int BM, int BN, int NS>
struct W16Tile {
  static constexpr int A = BM * 128, W = BN * 32, RUNS = (BN + 127) / 128;
  static constexpr int OFF_S = A + W, SLOT = OFF_S + 1024;
  static constexpr int OUT = BM * BN * 2;
  static constexpr int RING = NS * SLOT > OUT ? NS * SLOT : OUT;
  static constexpr int DMA_A = BM / 32, DMA_W = BN / 128, DMA = DMA_A + DMA_W + 1;
};

template <bool F16, int BM, int BN, int WGM, int NS>
__global__ void __launch_bounds__(256, 2) nvfp4_w16_pipe(const GemmParams p) {
  using L = W16Tile<BM, BN, NS>;
  constexpr int WGN = 4 / WGM, WM = BM / WGM, WN = BN / WGN, MB = WM / 32, NB = WN / 32;
  static_assert(WM % 32 == 0 && WN % 32 == 0 && BN % 128 == 0 && L::RUNS <= 2 && NS >= 3 && (NS - 1) * L::DMA < 64 &&
                2 * (L::RING + VEC_LDS) <= 160 * 1024, "tiling");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[L::RING];
  __shared__ __attribute__((aligned(1024))) uint8_t vec[VEC_LDS];
  int tm, tn;
  tile_coords((int)((p.m + BM - 1) / BM), (int)((p.n + BN - 1) / BN), p.group_m, tm, tn);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = (int)threadIdx.x & 63;
  const int wm = wave % WGM, wn = wave / WGM;
  const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int64_t rows_a = min((int64_t)BM, p.m - m0), rows_w = min((int64_t)BN, p.n - n0);
  const int64_t k_tiles = p.k / 64;
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a + m0 * p.lda, (uint32_t)(rows_a * p.lda));
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + n0 * p.ldw, (uint32_t)(rows_w * p.ldw));
  const __amdgpu_buffer_rsrc_t rs =
      make_rsrc(p.wsb + n0 / 128 * k_tiles * 512, (uint32_t)(rows_w / 128 * k_tiles * 512));
  const int KT = (int)k_tiles;

  const int drow = lane >> 3;
  const int ach0 = (lane & 7) ^ lds_swizzle(drow), ach1 = (lane & 7) ^ lds_swizzle(drow + 8);
  const uint32_t a_base0 = (uint32_t)((wave * (BM / 4) + drow) * p.lda + ach0 * 16);
  const uint32_t a_base1 = (uint32_t)((wave * (BM / 4) + drow + 8) * p.lda + ach1 * 16);
  const uint32_t a_step = (uint32_t)(16 * p.lda);
  // Packed rows of two chunks: chunk c of row r lies in slot c ^ ((r >> 3) & 1).
  const int wrow = lane >> 1, wch = (lane & 1) ^ ((wrow >> 3) & 1);
  const uint32_t w_base = (uint32_t)((wave * (BN / 4) + wrow) * p.ldw + wch * 16);
  const uint32_t w_step = (uint32_t)(32 * p.ldw);
  // Every wave copies the stage's scales, lanes 32-63 those of the second 128 rows.
  const uint32_t s_base = lane < 32 * L::RUNS ? (uint32_t)((lane >> 5) * k_tiles * 512 + (lane & 31) * 16) : VFA_OOB;
  auto issue = [&](int j, int s) {
    const uint32_t slot = ring_lds + (uint32_t)j * L::SLOT;
    const uint32_t kill = s < KT ? 0u : VFA_OOB;
    static_for<L::DMA_A>([&](auto i) {
      lds_dma16(ra, slot + wave * (L::A / 4) + i * 1024,
                ((i % 2 ? a_base1 : a_base0) + (i / 2) * a_step + (uint32_t)s * 128u) | kill);
    });
    static_for<L::DMA_W>([&](auto i) {
      lds_dma16(rw, slot + L::A + wave * (L::W / 4) + i * 1024, (w_base + i * w_step + (uint32_t)s * 32u) | kill);
    });
    lds_dma16(rs, slot + L::OFF_S, (s_base + (uint32_t)s * 512u) | kill | (s_base & VFA_OOB));
  };
  const int fr = lane & 31, fh = lane >> 5, asw = lds_swizzle(fr), wsw = (fr >> 3) & 1;
  v16f acc[NB][MB];
  static_for<NB>([&](auto i) { static_for<MB>([&](auto jj) { acc[i][jj] = v16f{}; }); });
  stage_vectors<BM, BN>(p, m0, n0, wave, lane, __builtin_amdgcn_readfirstlane(lds_addr(vec)));
  static_for<NS - 1>([&](auto s) { issue((int)s, (int)s); });
  auto stage = [&](int kt, auto jc) {
    constexpr int j = jc;
    wait_vmcnt<(NS - 2) * L::DMA, false>();  // stage kt, and before it the vectors
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();  // for every wave, which have all read stage kt - 1
    asm volatile("" ::: "memory");
    issue((j + NS - 1) % NS, kt + NS - 1);
    const uint8_t* base = ring + j * L::SLOT;
    v4i w[NB];
    uint32_t sw[NB];
    static_for<NB>([&](auto nb) {
      const int r = wn * WN + nb * 32;
      w[nb] = *reinterpret_cast<const v4i*>(base + L::A + (r + fr) * 32 + ((fh ^ wsw) << 4));
      sw[nb] = *reinterpret_cast<const uint32_t*>(base + L::OFF_S + r / 128 * 512 + fr * 16 + r % 128 / 32 * 4) >> (16 * fh);
    });
    static_for<4>([&](auto v) {
      v4i a[MB];
      static_for<MB>([&](auto mb) {
        a[mb] = *reinterpret_cast<const v4i*>(base + (wm * WM + mb * 32 + fr) * 128 + (((4 * fh + v) ^ asw) << 4));
      });
      static_for<NB>([&](auto nb) {
        const W16Scales<F16> s(sw[nb]);
        const v4i o = w16_restore<F16, v / 2>((uint32_t)w[nb][(int)v], s);
        static_for<MB>([&](auto mb) { acc[nb][mb] = w16_mfma32<F16>(o, a[mb], acc[nb][mb]); });
      });
    });
  };
  for (int kt = 0; kt < KT; kt += NS)
    static_for<NS>([&](auto i) {
      if (kt + i < KT) stage(kt + i, i);
    });
  wait_vmcnt<0, true>();  // every DMA has landed before the ring becomes the staging tile
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  const float alpha = *p.sw;
  static_for<NB>([&](auto nb) { static_for<MB>([&](auto mb) { acc[nb][mb] *= alpha; }); });
  gemm_epilogue<BM, BN, WGM, WGN, EPI_LINEAR, true, true>(p, acc, m0, n0, wm, wn, (int)threadIdx.x, ring, vec);
}

int compute_units();

namespace {

template <bool F16, int NB, int MB, int D>
void launch_few(const GemmParams& p, hipStream_t s) {
  const int64_t blocks_m = (p.m + 16 * MB - 1) / (16 * MB);
  const int64_t tiles = (p.n / 128 + 7) / 8 * 8;
  nvfp4_w16_few<F16, NB, MB, D><<<dim3((unsigned)(tiles * (8 / NB) * blocks_m)), dim3(512), 0, s>>>(p, (int)blocks_m);
}

template <bool F16, int BM, int BN, int WGM, int NS>
void launch_tile(const GemmParams& p, hipStream_t s) {
  const int64_t tiles = ((p.m + BM - 1) / BM) * ((p.n + BN - 1) / BN);
  nvfp4_w16_pipe<F16, BM, BN, WGM, NS><<<dim3((unsigned)tiles), dim3(256), 0, s>>>(p);
}

template <bool F16>
void launch_w16(const GemmParams& p, hipStream_t s) {
  const int64_t cus = compute_units();
  if (p.m <= 16) {
    if (p.n / 64 >= cus) launch_few<F16, 4, 1, 2>(p, s);
    else launch_few<F16, 1, 1, 4>(p, s);
  } else if (p.m <= 32) {
    launch_few<F16, 4, 2, 2>(p, s);
  } else if (p.m <= 256) {
    launch_few<F16, 4, 4, 2>(p, s);
  } else {
    launch_tile<F16, 128, 256, 1, 3>(p, s);
  }
}

}  // namespace

// a: x as bytes, lda its row stride in bytes.
hipError_t launch_nvfp4_w16(const GemmParams& params, bool f16, hipStream_t s) {
  GemmParams p = params;
  p.group_m = 8;
  if (f16) launch_w16<true>(p, s);
  else launch_w16<false>(p, s);
  return hipGetLastError();
}

}  // namespace vfa
