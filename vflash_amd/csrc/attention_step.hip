// Packed attention for gfx950: tiles of up to 16 rows (a token or a few per sequence).
//
// Bound by the bytes of K and V, each read once per key head.  The products are those of
// attention.hip with v_mfma_f32_16x16x32: S^T = K Q^T for 16 keys at a time, O^T = V^T P^T for 32,
// where K position (lane row g, j) stands for key 4 g + j of the first 16 keys (j < 4) or
// 4 g + j - 4 of the second, which is where the scores lie.
//
// Each wave takes every fourth block of 32 keys of the item and keeps a ring of two in LDS, which
// its own DMA fills: 128 KB a CU in flight or in use, no barrier before the end, where the four
// waves' sums are added up.  131071 keys of 8 heads of 128: 107 us, 5.0 TB/s, what a copy of 1 GiB
// reaches; 16 sequences of up to 8191: 65 us, 4.2 TB/s; 77 keys: 7.5 us a call, a chain of loads, search
// and sums in one wave after another.
#include "attention.h"

namespace vfa {

template <int DP>
struct AttentionSteps {
  static constexpr int PITCH = DP <= 64 ? 128 : 256, CHUNKS = PITCH / 16, ROWS = 1024 / PITCH;
  static constexpr int KEYS = 32, TILE = KEYS * PITCH, SLOT = 2 * TILE, NS = 2, WAVES = 4;
  static constexpr int DMA = SLOT / 1024;  // instructions per stage
  static constexpr int ACC = DP * 4 + 16;  // bytes of a row's sums in LDS
};
template <int PITCH>
__device__ __forceinline__ int step_k_swizzle(int r) {
  return PITCH == 256 ? r & 15 : lds_swizzle(r);
}
// Eight rows x two chunks of a half wave's transposing read take different slots.
template <int PITCH>
__device__ __forceinline__ int step_v_swizzle(int r) {
  return PITCH == 256 ? (r & 7) << 1 : (r >> 1 & 3) << 1;
}

template <bool F16, int DP>
__global__ void __launch_bounds__(256, 1) attention_step(const AttentionParams p) {
  using L = AttentionSteps<DP>;
  constexpr int QS = (DP + 31) / 32, DB = DP / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[L::WAVES * L::NS * L::SLOT];
  __shared__ float stat[L::WAVES][16][2];
  static_assert(L::WAVES * 16 * L::ACC <= L::WAVES * L::NS * L::SLOT && (L::NS - 1) * L::DMA < 64, "LDS, vmcnt");
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = (int)threadIdx.x & 63;
  const int fr = lane & 15, fg = lane >> 4;
  uint8_t* ring = lds + wave * (L::NS * L::SLOT);
  const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));

  const AttentionLine line = attention_line(p, gridDim.x);
  const uint32_t begin = (blockIdx.x >> (line.xcds == 8 ? 3 : 0)) * line.quota, stop = min(begin + line.quota, line.end);
  for (uint32_t pos = begin; pos < stop;) {
    const AttentionSegment seg = attention_segment(p, line, blockIdx.x, pos, stop);
    const AttentionItem& it = seg.it;
    if (!it.live) return;
    const AttentionRow row = attention_row(p, it, fr);
    const int key_head = attention_key_head(p, it.head_block);
    const int last_token = min(it.seq.nq, (it.tile + 1) * p.tile_tokens) - 1;
    const int tile_limit = attention_limit(p, it.seq, last_token);
    const int first = (int)min((uint64_t)seg.first << line.unit_shift, (uint64_t)INT32_MAX);
    const int last = (int)min((uint64_t)tile_limit, (uint64_t)(seg.first + seg.count) << line.unit_shift);
    const int limit = row.live ? min(attention_limit(p, it.seq, row.token), last) : last;
    // Keys that every row sees.
    const int open = min(attention_limit(p, it.seq, min(it.tile * p.tile_tokens, it.seq.nq)), last);

    const uint8_t* kb = reinterpret_cast<const uint8_t*>(p.k + (int64_t)it.seq.k0 * p.k_ts + (int64_t)key_head * p.k_hs);
    const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.v + (int64_t)it.seq.k0 * p.v_ts + (int64_t)key_head * p.v_hs);
    const uint32_t kts = (uint32_t)p.k_ts * 2, vts = (uint32_t)p.v_ts * 2;
    const int drow = lane / L::CHUNKS, dslot = lane % L::CHUNKS;
    auto issue = [&](int buf, int key0) {
      const int left = last - key0;  // none: every lane reads zeros
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(kb + (int64_t)key0 * kts, 0x7fffffffu);
      const __amdgpu_buffer_rsrc_t rv = make_rsrc(vb + (int64_t)key0 * vts, 0x7fffffffu);
      const uint32_t dst = ring_lds + buf * L::SLOT;
      static_for<L::DMA / 2>([&](auto i) {
        const int r = drow + i * L::ROWS;
        const int c = dslot ^ step_k_swizzle<L::PITCH>(r);
        lds_dma16(rk, dst + i * 1024, r < left && c * 8 < p.dim ? (uint32_t)r * kts + c * 16 : VFA_OOB);
      });
      static_for<L::DMA / 2>([&](auto i) {
        const int r = drow + i * L::ROWS;
        const int c = dslot ^ step_v_swizzle<L::PITCH>(r);
        lds_dma16(rv, dst + L::TILE + i * 1024, r < left && c * 8 < p.dim ? (uint32_t)r * vts + c * 16 : VFA_OOB);
      });
    };
    constexpr int STRIDE = L::WAVES * L::KEYS;
    const int start = first + wave * L::KEYS;
    static_for<L::NS>([&](auto i) { issue(i, start + i * STRIDE); });

    v4i q[QS];
    static_for<QS>([&](auto s) { q[s] = attention_query(p, it, row, s * 32 + fg * 8); });
    v4f o[DB];
    static_for<DB>([&](auto i) { o[i] = v4f{}; });
    float m = VFA_LOWEST, l = 0;
    bool far = false;
    const uint8_t* krow = ring + fr * L::PITCH;
    const int ksw = step_k_swizzle<L::PITCH>(fr);
    const int vr = 4 * fg + ((lane >> 2) & 3);
    const int vc = (lane & 3) >> 1;
    const uint8_t* vrow = ring + L::TILE + vr * L::PITCH + (lane & 1) * 8;
    const int vsw = step_v_swizzle<L::PITCH>(vr);

    int buf = 0;
    for (int key0 = start; key0 < last; key0 += STRIDE, buf = buf + 1 == L::NS ? 0 : buf + 1) {
      wait_vmcnt<(L::NS - 1) * L::DMA, false>();
      asm volatile("" ::: "memory");
      v4f s[2];
      static_for<2>([&](auto kbk) {
        s[kbk] = v4f{};
        static_for<QS>([&](auto st) {
          const v4i a = *reinterpret_cast<const v4i*>(krow + buf * L::SLOT + kbk * 16 * L::PITCH +
                                                      (((4 * st + fg) ^ ksw) << 4));
          s[kbk] = mfma16<F16>(a, q[st], s[kbk]);
        });
      });
      if (key0 + L::KEYS > open) {
        const int lim = limit - key0 - 4 * fg;
        static_for<2>([&](auto kbk) {
          static_for<4>([&](auto r) { s[kbk][(int)r] = kbk * 16 + r < lim ? s[kbk][(int)r] : -__builtin_inff(); });
        });
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = max_across32(max_across16(mx));
      if (__builtin_amdgcn_ballot_w64(mx * p.c > m * p.c + kAttentionSlack)) {
        const float next = fmaxf(m, mx), f = __builtin_amdgcn_exp2f((m - next) * p.c);
        static_for<DB>([&](auto i) { static_for<4>([&](auto r) { o[i][(int)r] *= f; }); });
        l *= f;
        m = next;
        far = __builtin_amdgcn_ballot_w64(fabsf(m * p.c) >= kAttentionFar && m > VFA_LOWEST) != 0;
      }
      const float ref = attention_shift<F16>(p) - attention_top(m, p.c);
      v4i pk;
      auto weights = [&](auto far_rows) {
        static_for<4>([&](auto j) {
          constexpr int r = (j % 2) * 2;
          pk[(int)j] = pack2<F16>(attention_weight<far_rows>(s[j / 2][r], p.c, m, ref, attention_shift<F16>(p)),
                                  attention_weight<far_rows>(s[j / 2][r + 1], p.c, m, ref, attention_shift<F16>(p)));
          l = attention_sum2<F16>(pk[(int)j], l);
        });
      };
      if (far) weights(std::true_type{});
      else weights(std::false_type{});
      static_for<DB>([&](auto db) {
        const uint8_t* src = vrow + buf * L::SLOT + (((2 * db + vc) ^ vsw) << 4);
        const v2i lo = lds_read_tr16(src), hi = lds_read_tr16(src + 16 * L::PITCH);
        o[db] = mfma16<F16>(v4i{lo[0], lo[1], hi[0], hi[1]}, pk, o[db]);
      });
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot is read
      asm volatile("" ::: "memory");
      issue(buf, key0 + L::NS * STRIDE);
    }
    l = sum_across32(sum_across16(l));
    wait_vmcnt<0, true>();
    asm volatile("" ::: "memory");
    __syncthreads();  // every ring is done with
    static_for<DB>([&](auto db) {
      *reinterpret_cast<v4f*>(lds + (wave * 16 + fr) * L::ACC + (db * 16 + 4 * fg) * 4) = o[db];
    });
    if (fg == 0) {
      stat[wave][fr][0] = attention_top(m, p.c);
      stat[wave][fr][1] = l;
    }
    __syncthreads();
    // Thread t: row t / 16, the d of t % 16 in runs of four.
    const int r = (int)threadIdx.x >> 4, e = (int)threadIdx.x & 15;
    const AttentionRow mine = attention_row(p, it, r);
    if (mine.live) {
      float top = stat[0][r][0], sum = 0, f[L::WAVES];
      static_for<L::WAVES - 1>([&](auto w) { top = fmaxf(top, stat[w + 1][r][0]); });
      static_for<L::WAVES>([&](auto w) {
        f[w] = __builtin_amdgcn_exp2f(stat[w][r][0] - top);
        sum += f[w] * stat[w][r][1];
      });
      const bool whole = seg.count == seg.of;
      const int64_t at = (2 * (int64_t)blockIdx.x + (seg.first == 0)) * 16 + r;
      if (!whole && e == 0) *reinterpret_cast<v2f*>(p.part_ml + at * 2) = v2f{top, sum};
      const float inv = whole ? 1.0f / sum : 1.0f;
      uint16_t* dst = p.out + (int64_t)(it.seq.q0 + mine.token) * p.o_ts + (int64_t)mine.head * p.o_hs;
      for (int d = 4 * e; d < p.dim; d += 64) {
        v4f x = v4f{};
        static_for<L::WAVES>(
            [&](auto w) { x += *reinterpret_cast<const v4f*>(lds + (w * 16 + r) * L::ACC + d * 4) * f[w]; });
        x = sum == 0 ? v4f{} : x * inv;
        if (whole) *reinterpret_cast<v2i*>(dst + d) = v2i{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3])};
        else *reinterpret_cast<v4f*>(p.part + at * p.dim + d) = x;
      }
    }
    pos += seg.count;
    if (pos < stop) __syncthreads();  // the sums are read: the rings may be filled again
  }
}

// The sum over a tile's segments: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  Workgroup b
// takes the tile that workgroup b of attention_step began and did not end.  Thread t: d 4 (t % 16) and
// 64 more, one row, every groups-th segment under a maximum of its own; the groups meet in LDS.
template <bool F16>
__global__ void __launch_bounds__(1024) attention_step_join(const AttentionParams p) {
  const AttentionLine line = attention_line(p, gridDim.x);
  const int part = blockIdx.x >> (line.xcds == 8 ? 3 : 0);
  const uint32_t begin = part * line.quota, stop = min(begin + line.quota, line.end);
  if (begin >= stop) return;
  const AttentionSegment seg = attention_segment(p, line, blockIdx.x, stop - 1, line.end);
  const uint32_t tile_begin = stop - 1 - seg.first, tile_end = tile_begin + seg.of;
  if (!seg.it.live || tile_begin < begin || tile_end <= stop) return;
  const int segments = (int)((tile_end - 1) / line.quota) - part + 1;
  // Segment s lies in workgroup blockIdx.x + xcds s, slot 1 for the first, 0 for the others.
  auto slot = [&](int s) { return 2 * ((int64_t)blockIdx.x + line.xcds * s) + (s == 0); };
  const int tokens = min(p.tile_tokens, seg.it.seq.nq - seg.it.tile * p.tile_tokens);
  const int rows = min(16, tokens * p.heads_per_tile);
  const int pow = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  const int groups = min(16, 64 / pow);
  const int e = (int)threadIdx.x & 15, r = (int)threadIdx.x / 16 % pow, sg = (int)threadIdx.x / 16 / pow;
  __shared__ float sums[64][132];
  float top = VFA_LOWEST, l = 0;
  v4f x[2] = {v4f{}, v4f{}};
#pragma unroll 4
  for (int s = sg; s < segments && sg < groups; s += groups) {
    const int64_t at = slot(s) * 16 + r;
    const v2f ml = *reinterpret_cast<const v2f*>(p.part_ml + at * 2);
    const float next = fmaxf(top, ml[0]);
    const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(ml[0] - next);
    top = next;
    l = l * old + f * ml[1];
    static_for<2>([&](auto h) {
      const int d = 4 * e + 64 * h;
      if (d < p.dim) x[h] = x[h] * old + *reinterpret_cast<const v4f*>(p.part + at * p.dim + d) * f;
    });
  }
  float* mine = sums[(int)threadIdx.x / 16];
  static_for<2>([&](auto h) { *reinterpret_cast<v4f*>(mine + 4 * e + 64 * h) = x[h]; });
  if (e == 0) {
    mine[128] = l;
    mine[129] = top;
  }
  __syncthreads();
  const AttentionRow row = attention_row(p, seg.it, r);
  if (sg || !row.live) return;
  float all = top;
  for (int q = 1; q < groups; ++q) all = fmaxf(all, sums[q * pow + r][129]);
  const float f0 = __builtin_amdgcn_exp2f(top - all);
  l *= f0;
  static_for<2>([&](auto h) { x[h] *= f0; });
  for (int q = 1; q < groups; ++q) {
    const float* other = sums[q * pow + r];
    const float f = __builtin_amdgcn_exp2f(other[129] - all);
    static_for<2>([&](auto h) { x[h] += *reinterpret_cast<const v4f*>(other + 4 * e + 64 * h) * f; });
    l += other[128] * f;
  }
  const float inv = 1.0f / l;
  uint16_t* dst = p.out + (int64_t)(seg.it.seq.q0 + row.token) * p.o_ts + (int64_t)row.head * p.o_hs;
  static_for<2>([&](auto h) {
    const int d = 4 * e + 64 * h;
    const v4f y = l == 0 ? v4f{} : x[h] * inv;
    if (d < p.dim) *reinterpret_cast<v2i*>(dst + d) = v2i{pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3])};
  });
}

void launch_attention_step(const AttentionParams& p, bool f16, int grid, bool join, hipStream_t s) {
  const dim3 g((unsigned)grid), b(256);
  if (p.dim <= 64) {
    if (f16) attention_step<true, 64><<<g, b, 0, s>>>(p);
    else attention_step<false, 64><<<g, b, 0, s>>>(p);
  } else {
    if (f16) attention_step<true, 128><<<g, b, 0, s>>>(p);
    else attention_step<false, 128><<<g, b, 0, s>>>(p);
  }
  if (!join) return;
  if (f16) attention_step_join<true><<<g, dim3(1024), 0, s>>>(p);
  else attention_step_join<false><<<g, dim3(1024), 0, s>>>(p);
}

}  // namespace vfa
