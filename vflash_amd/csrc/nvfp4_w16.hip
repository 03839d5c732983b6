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

// The eight values of packed word d times their block scale, as an MFMA operand.
template <bool F16>
__device__ __forceinline__ v4i w16_restore(uint32_t d, float s) {
  v4i o;
  static_for<4>([&](auto i) {
    if constexpr (F16) {
      const _Float16 h = (_Float16)s;  // exact, as every E4M3 value
      o[(int)i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, 1.0f, (int)i) * v2hf{h, h});
    } else {
      const v2f y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, (int)i);
      const float a = y[0] * s, b = y[1] * s;
      o[(int)i] = (int)pack_bf16x2(a, b);
    }
  });
  return o;
}

// ---------------------------------------------------------------------------
// Few rows.  A workgroup computes 16 MB rows of x times 16 NB rows of the weight.  Its waves take
// every WAVES-th stage of KS K each, through an LDS ring of their own that DMA fills NS stages
// ahead, with no barrier before the end, where the waves' sums meet.  Loads straight into the
// operands' lane order would do without LDS, but neighbouring lanes hold different rows there: at an
// access per 16 bytes the vector cache alone took 20 us of the 31 that 64 x 5120 x 15360 then took.
// The 16-row blocks of a workgroup lie 32 rows apart, as the scales of one 16-byte run do.
//
// Bound by the weight's bytes from one row to a few where it is large (1 x 5376 x 28672 in f16 16.7 us,
// 5.2 TB/s), by one launch's latency where it is small (1 x 5120 x 5120 6.9), and at 64 rows by x,
// which every workgroup takes through L2 and LDS (64 x 5120 x 15360 20.6, 2.3 TB/s of all bytes).
//
// Lane group g takes K g KS / 4 .. of a stage, so that it reads its packed values at once: step v of
// 32 K multiplies K g KS / 4 + 8 v .. + 7 of each group.
template <int NB, int MB, int XR, int KS, int WAVES, int NS>
struct W16Few {
  static constexpr int WROW = KS / 2, XROW = 2 * KS;                  // bytes of a row's stage
  static constexpr int W = 16 * NB * WROW, X = XR * XROW, S = KS / 64 * 256;
  static constexpr int STAGE = W + X + S, RING = NS * STAGE;
  static constexpr int DMA_W = (W + 1023) / 1024, DMA_X = X / 1024, DMA = DMA_W + DMA_X + 1;
  static constexpr int PITCH = 16 * NB + 4, SUMS = WAVES * 16 * MB * PITCH * 4;
  static constexpr int LDS = WAVES * RING > SUMS ? WAVES * RING : SUMS;
  static constexpr int STEPS = KS / 32;
  static_assert(X % 1024 == 0 && (NS - 1) * DMA < 64 && LDS <= 160 * 1024, "stages");
};

template <bool F16, int NB, int MB, int XR, int KS, int WAVES, int NS>
__global__ void __launch_bounds__(64 * WAVES) nvfp4_w16_few(const GemmParams p, int blocks_m) {
  using L = W16Few<NB, MB, XR, KS, WAVES, NS>;
  constexpr int SUBS = 8 / NB;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[L::LDS];
  // The workgroups of a 128-row tile and a block of x rows run on one XCD, whose L2 then serves the
  // scales and x rows that they share; the tiles and blocks go round the XCDs.
  const int xcd = (int)blockIdx.x & 7, j = (int)blockIdx.x >> 3;
  const int64_t group = (int64_t)(j / SUBS) * 8 + xcd, n_tiles = p.n / 128;
  if (group >= n_tiles * blocks_m) return;
  const int sub = j % SUBS;
  const int64_t block = group / n_tiles, tile = group - block * n_tiles;
  const int64_t m0 = block * (16 * MB);
  const int half = sub & 1, b0 = (sub >> 1) * NB;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = (int)threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int k_tiles = (int)(p.k / 64), stages = (int)((p.k + KS - 1) / KS);
  const int rows = (int)min((int64_t)(16 * MB), p.m - m0);
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + (tile * 128 + 32 * b0 + 16 * half) * p.ldw, 0x7fffffffu);
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.wsb + (tile * k_tiles * 512 + 256 * half), 0x7fffffffu);
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.a + m0 * p.lda, 0x7fffffffu);
  uint8_t* ring = lds + wave * L::RING;
  const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));

  // 16-byte chunk c of row r lies in slot c ^ key(r), so that the reads of 16 rows meet no bank twice.
  constexpr int WCH = L::WROW / 16, XCH = L::XROW / 16;
  auto w_key = [](int r) { return KS == 128 ? (r >> 2) & 3 : (r >> 3) & 1; };
  auto x_key = [](int r) { return KS == 128 ? r & 15 : lds_swizzle(r); };
  // Stage s (past the last one: nothing is read) into slot j.
  auto issue = [&](int j, int s) {
    const uint32_t dst = ring_lds + j * L::STAGE;
    const int left = (int)p.k - s * KS;  // K
    static_for<L::DMA_W>([&](auto q) {
      const int r = q * (64 / WCH) + lane / WCH, c = (lane % WCH) ^ w_key(r & 15);  // r: 16 b + i
      const uint32_t off = (uint32_t)((r >> 4) * 32 + (r & 15)) * (uint32_t)p.ldw + (uint32_t)s * L::WROW + c * 16;
      if (L::W % 1024 == 0 || lane < L::W % 1024 / 16) lds_dma16(rw, dst + q * 1024, c * 32 < left ? off : VFA_OOB);
    });
    static_for<L::DMA_X>([&](auto q) {
      const int r = q * (64 / XCH) + lane / XCH, c = (lane % XCH) ^ x_key(r);
      const uint32_t off = (uint32_t)r * (uint32_t)p.lda + (uint32_t)s * L::XROW + c * 16;
      lds_dma16(rx, dst + L::W + q * 1024, c * 8 < left && r < rows ? off : VFA_OOB);
    });
    if (lane < KS / 64 * 16)
      lds_dma16(rs, dst + L::W + L::X,
                (lane >> 4) * 64 < left ? (uint32_t)(s * (KS / 64) + (lane >> 4)) * 512 + (lane & 15) * 16 : VFA_OOB);
  };
  v4f acc[NB][MB];
  static_for<NB>([&](auto b) { static_for<MB>([&](auto m) { acc[b][m] = v4f{}; }); });
  static_for<NS>([&](auto q) { issue(q, wave + WAVES * q); });
  int slot = 0;
  for (int s = wave; s < stages; s += WAVES, slot = slot + 1 == NS ? 0 : slot + 1) {
    wait_vmcnt<(NS - 1) * L::DMA, false>();
    asm volatile("" ::: "memory");
    const uint8_t* base = ring + slot * L::STAGE;
    uint32_t w[NB][L::STEPS];
    float sc[NB][(L::STEPS + 1) / 2];
    static_for<NB>([&](auto b) {
      const uint8_t* row = base + (16 * b + i) * L::WROW;
      if constexpr (KS == 128) {
        const v4i q = *reinterpret_cast<const v4i*>(row + ((g ^ w_key(i)) << 4));
        static_for<4>([&](auto v) { w[b][v] = (uint32_t)q[(int)v]; });
        const uint32_t word = *reinterpret_cast<const uint32_t*>(base + L::W + L::X + (g >> 1) * 256 + i * 16 + 4 * (b0 + b));
        const v2f y = __builtin_amdgcn_cvt_pk_f32_fp8((int)(word >> (16 * (g & 1))), false);
        sc[b][0] = y[0];
        sc[b][1] = y[1];
      } else {
        const uint2 q = *reinterpret_cast<const uint2*>(row + (((g >> 1) ^ w_key(i)) << 4) + 8 * (g & 1));
        w[b][0] = q.x;
        w[b][1] = q.y;
        const uint32_t word = *reinterpret_cast<const uint32_t*>(base + L::W + L::X + i * 16 + 4 * (b0 + b));
        sc[b][0] = __builtin_amdgcn_cvt_f32_fp8((int)(word >> (8 * g)), 0);
      }
    });
    static_for<L::STEPS>([&](auto v) {
      v4i x[MB];
      static_for<MB>([&](auto m) {
        const int r = (16 * m + i) % XR;  // rows past XR: columns of the product that nobody reads
        x[m] = *reinterpret_cast<const v4i*>(base + L::W + r * L::XROW + (((g * L::STEPS + v) ^ x_key(r)) << 4));
      });
      static_for<NB>([&](auto b) {
        const v4i o = w16_restore<F16>(w[b][v], sc[b][v / 2]);
        static_for<MB>([&](auto m) { acc[b][m] = mfma16<F16>(o, x[m], acc[b][m]); });
      });
    });
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot is read
    asm volatile("" ::: "memory");
    issue(slot, s + WAVES * NS);
  }
  wait_vmcnt<0, true>();
  asm volatile("" ::: "memory");
  __syncthreads();  // every ring is done with
  float* sums = reinterpret_cast<float*>(lds);
  // Lane (m, g) holds the weight rows 4 g .. + 3 of its blocks.
  static_for<NB>([&](auto b) {
    static_for<MB>([&](auto m) {
      *reinterpret_cast<v4f*>(sums + (wave * 16 * MB + 16 * m + i) * L::PITCH + 16 * b + 4 * g) = acc[b][m];
    });
  });
  __syncthreads();
  const float alpha = *p.sw;
  for (int e = (int)threadIdx.x; e < 16 * MB * 4 * NB; e += 64 * WAVES) {
    const int m = e / (4 * NB), c = e % (4 * NB) * 4;
    if (m >= rows) break;
    v4f y = v4f{};
    static_for<WAVES>([&](auto w) { y += *reinterpret_cast<const v4f*>(sums + (w * 16 * MB + m) * L::PITCH + c); });
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
// wide, so that none restores another's weights; 1021 x 5120 x 13824 126 us, 1.15 PFLOP/s on a grid that
// fills 84 % of its two rounds.  Each of a stage's four steps multiplies while the
// next one's operands are read and restored between its MFMAs.
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
  struct Raw {
    v4i w[NB];
    uint32_t s[NB];
  };
  struct Step {
    v4i w[NB], a[MB];
  };
  auto read_w = [&](Raw& r, const uint8_t* base) {
    static_for<NB>([&](auto nb) {
      const int n = wn * WN + nb * 32;
      r.w[nb] = *reinterpret_cast<const v4i*>(base + L::A + (n + fr) * 32 + ((fh ^ wsw) << 4));
      r.s[nb] = *reinterpret_cast<const uint32_t*>(base + L::OFF_S + n / 128 * 512 + fr * 16 + n % 128 / 32 * 4);
    });
  };
  auto read_a = [&](Step& o, const uint8_t* base, auto v) {
    static_for<MB>([&](auto mb) {
      o.a[mb] = *reinterpret_cast<const v4i*>(base + (wm * WM + mb * 32 + fr) * 128 + (((4 * fh + v) ^ asw) << 4));
    });
  };
  auto restore = [&](Step& o, const Raw& r, auto v) {
    static_for<NB>([&](auto nb) {
      const float s = __builtin_amdgcn_cvt_f32_fp8((int)(r.s[nb] >> (16 * fh)), v / 2);
      o.w[nb] = w16_restore<F16>((uint32_t)r.w[nb][(int)v], s);
    });
  };
  // One step's MFMAs with the next step's conversions between them.
  constexpr int VALU = (F16 ? 10 : 18) * NB / (NB * MB) + 1;
  auto multiply = [&](const Step& o) {
    static_for<NB>([&](auto nb) {
      static_for<MB>([&](auto mb) { acc[nb][mb] = mfma32<F16>(o.w[nb], o.a[mb], acc[nb][mb]); });
    });
    static_for<NB * MB>([&](auto) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    });
    __builtin_amdgcn_sched_barrier(0);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  stage_vectors<BM, BN>(p, m0, n0, wave, lane, __builtin_amdgcn_readfirstlane(lds_addr(vec)));
  static_for<NS - 1>([&](auto s) { issue((int)s, (int)s); });
  wait_vmcnt<(NS - 2) * L::DMA, false>();  // stage 0, and before it the vectors
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Raw raw[2];
  Step st[2];
  read_w(raw[0], ring);
  read_a(st[0], ring, I0{});
  restore(st[0], raw[0], I0{});
  auto stage = [&](int kt, auto jc, auto par) {
    constexpr int j = jc;
    const uint8_t* base = ring + j * L::SLOT;
    const uint8_t* next = ring + (j + 1) % NS * L::SLOT;
    Raw &r = raw[par], &rn = raw[1 - par];
    read_a(st[1], base, I1{});
    restore(st[1], r, I1{});
    multiply(st[0]);
    read_a(st[0], base, I2{});
    restore(st[0], r, I2{});
    multiply(st[1]);
    // Stage kt + 1 has landed for every wave, and every wave has read stage kt - 1, whose slot
    // takes stage kt + NS - 1.
    wait_vmcnt<(NS - 3) * L::DMA, false>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue((j + NS - 1) % NS, kt + NS - 1);
    read_w(rn, next);  // zeros past the last stage, never multiplied
    read_a(st[1], base, I3{});
    restore(st[1], r, I3{});
    multiply(st[0]);
    read_a(st[0], next, I0{});
    restore(st[0], rn, I0{});
    multiply(st[1]);
  };
  constexpr int TRIP = NS % 2 ? 2 * NS : NS;  // slot and register set are constants of a stage
  for (int kt = 0; kt < KT; kt += TRIP)
    static_for<TRIP>([&](auto i) {
      if (kt + i < KT) stage(kt + i, std::integral_constant<int, i % NS>{}, std::integral_constant<int, i % 2>{});
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

template <bool F16, int NB, int MB, int XR, int KS, int WAVES, int NS>
void launch_few(const GemmParams& p, hipStream_t s) {
  const int64_t blocks_m = (p.m + 16 * MB - 1) / (16 * MB);
  const int64_t groups = (p.n / 128 * blocks_m + 7) / 8 * 8;
  nvfp4_w16_few<F16, NB, MB, XR, KS, WAVES, NS>
      <<<dim3((unsigned)(groups * (8 / NB))), dim3(64 * WAVES), 0, s>>>(p, (int)blocks_m);
}

template <bool F16, int BM, int BN, int WGM, int NS>
void launch_tile(const GemmParams& p, hipStream_t s) {
  const int64_t tiles = ((p.m + BM - 1) / BM) * ((p.n + BN - 1) / BN);
  nvfp4_w16_pipe<F16, BM, BN, WGM, NS><<<dim3((unsigned)tiles), dim3(256), 0, s>>>(p);
}

// Tiles of 64 x 64 (the few-row kernel) or 128 x 256, by the time of the busiest CU: 19 us a round of
// the first at K = 5120 (128 x 5120 x 5120, 160 workgroups 20.9; 300 rows, 400 workgroups 38.8) and 64
// of the second (300 rows, 60 tiles 65; 1021 x 5120 x 13824, 432 tiles 126), in proportion to K.  A
// round takes as long where it fills part of the CUs: 64 x 5120 x 5120, 80 workgroups, 19.6.
bool many_rows(int64_t m, int64_t n, int64_t cus) {
  const int64_t few = (m + 63) / 64 * (n / 64), many = (m + 127) / 128 * ((n + 255) / 256);
  return 64 * ((many + cus - 1) / cus) < 19 * ((few + cus - 1) / cus);
}

template <bool F16>
void launch_w16(const GemmParams& p, hipStream_t s) {
  const int64_t cus = compute_units();
  // Up to 16 rows a workgroup takes 64 weight rows where these fill the GPU and 32 where not:
  // 1 x 5120 x 5120 7.7 us with 160 workgroups of 32 rows and twice the waves, 10.5 with 80 of 64 rows,
  // and 1 x 5376 x 28672 17.9 us.  x in stages of four rows where it has no more: a quarter of its LDS.
  if (p.m <= 4) {
    if (p.n / 64 >= cus) launch_few<F16, 4, 1, 4, 128, 4, 2>(p, s);
    else launch_few<F16, 2, 1, 4, 128, 8, 4>(p, s);
  } else if (p.m <= 16) {
    if (p.n / 64 >= cus) launch_few<F16, 4, 1, 16, 128, 4, 2>(p, s);
    else launch_few<F16, 2, 1, 16, 128, 8, 3>(p, s);
  } else if (p.m <= 32) {
    launch_few<F16, 4, 2, 32, 64, 8, 2>(p, s);
  } else if (!many_rows(p.m, p.n, cus)) {
    launch_few<F16, 4, 4, 64, 64, 7, 2>(p, s);
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
