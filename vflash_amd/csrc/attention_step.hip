// Packed attention for gfx950: tiles of up to 16 rows (a token or a few per sequence).
//
// Bound by the bytes of K and V, each read once per key head.  The products are those of
// attention.hip with v_mfma_f32_16x16x32: S^T = K Q^T for 16 keys at a time, O^T = V^T P^T for 32,
// where K position (lane row g, j) stands for key 4 g + j of the first 16 keys (j < 4) or
// 4 g + j - 4 of the second, which is where the scores lie.
//
// Each of a workgroup's W waves takes every W-th block of 32 keys of the item and keeps a ring of NS blocks in
// LDS, which its own DMA fills: no barrier before the end, where the waves' sums are added up.  W is 4 over
// rows and wherever keys are split, 2 or 1 for many whole sequences over pages (the plan says which); NS is 2, but 1 for
// single waves of what is not E4M3 at dimension 128: these have one block each on its way, and overlap loads and
// products across the workgroups of a CU alone.  Four waves of two blocks of 16 bits hold 128 KB a CU in flight or in
// use: 131071 keys of 8 heads of 128 107 us, 5.0 TB/s, what a copy of 1 GiB reaches; 16 sequences of up
// to 8191: 63 us, 4.4 TB/s; 77 keys: 7.7 us a call, a chain of loads, search and sums in one wave after another.
//
// A paged cache differs in where a block's keys come from: each 16 lie in one page, whose number a scalar
// load fetches one block ahead.  E4M3 codes go to LDS as they are, with their factors, and become 16 bits between
// LDS and the matrix cores (exactly): a key's factor multiplies its score, a value's its weight before that is
// rounded, to bf16 whatever q's type (a factor has binary32's range); for f16 to two of it.
#include "attention_codes.h"

namespace vfa {

template <int DP, int STORE, int W>
struct AttentionSteps {
  static constexpr bool E4M3 = STORE == kStoreE4M3;
  static constexpr int PITCH = (DP <= 64 ? 64 : 128) * (E4M3 ? 1 : 2), CHUNKS = PITCH / 16, ROWS = 1024 / PITCH;
  static constexpr int KEYS = 32, TILE = KEYS * PITCH, SLOT = 2 * TILE + (E4M3 ? 512 : 0), WAVES = W;
  // One slot lets twice as many workgroups of one wave share a CU: 86 sequences of 4 keys, 56 heads of their own, in bf16
  // 18.4 us, with two 27.8, at dimension 64 12.0 and 15.5; in E4M3 at 128, of 128 keys, 43.5 and 37.8.
  static constexpr int NS = W == 1 && (DP <= 64 || !E4M3) ? 1 : 2;
  static constexpr int DMA = 2 * TILE / 1024 + (E4M3 ? 2 : 0);  // instructions per stage
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

// Tiles of codes: the 16 rows of a score block, and the eight rows of a transposing read (four keys from each
// half of the block), take different slots.
template <int PITCH>
__device__ __forceinline__ int step_k_code_swizzle(int r) {
  return PITCH == 128 ? r >> 1 & 7 : r >> 2 & 3;
}
template <int PITCH>
__device__ __forceinline__ int step_v_code_swizzle(int r) {
  return PITCH == 128 ? (r >> 1 & 3) | (r >> 4 & 1) << 2 : (r >> 2 & 1) | (r >> 4 & 1) << 1;
}

// Eight bytes per lane, transposed inside each group of 16 lanes: lanes 2 r and 2 r + 1 give the address of
// elements 0 .. 7 and 8 .. 15 of row r, and lane i receives element i of the eight rows.
__device__ __forceinline__ v2i lds_read_tr8(const uint8_t* p) {
  typedef __attribute__((address_space(3))) v2i lds_v2i;
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(uint32_t)lds_addr(p));
}
// lds_dma16 with four bytes a lane.
__device__ __forceinline__ void lds_dma4(__amdgpu_buffer_rsrc_t r, uint32_t lds_dst, uint32_t voffset) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds_dst), "v"(voffset), "s"(r)
               : "m0");
}

// E4M3 at dimension 64: four workgroups a CU.
template <bool F16, int DP, int STORE, int W>
__global__ void __launch_bounds__(64 * W, STORE == kStoreE4M3 && DP <= 64 ? 4 : 1) attention_step(const AttentionParams p) {
  using L = AttentionSteps<DP, STORE, W>;
  constexpr bool PAGED = STORE != kStoreRows, E4M3 = L::E4M3;
  constexpr bool W16 = F16 && !E4M3;  // the type of the weights
  constexpr int QS = (DP + 31) / 32, DB = DP / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[L::WAVES * L::NS * L::SLOT];
  __shared__ float stat[L::WAVES][16][2];
  static_assert(L::WAVES * 16 * L::ACC <= L::WAVES * L::NS * L::SLOT && (L::NS - 1) * L::DMA < 64, "LDS, vmcnt");
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = (int)threadIdx.x & 63;
  const int fr = lane & 15, fg = lane >> 4;
  uint8_t* ring = lds + wave * (L::NS * L::SLOT);
  const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_addr(ring));

  const AttentionLine line = attention_line<PAGED>(p, gridDim.x);
  const uint32_t begin = (blockIdx.x >> (line.xcds == 8 ? 3 : 0)) * line.quota, stop = min(begin + line.quota, line.end);
  [[maybe_unused]] AttentionSegment ended{};  // the last
  for (uint32_t pos = begin; pos < stop;) {
    const AttentionSegment seg = [&] {
      if constexpr (PAGED)
        return attention_scalar(pos == begin ? attention_segment<true>(p, line, blockIdx.x, pos, stop)
                                             : attention_following<true>(p, line, blockIdx.x, ended, pos, stop));
      else
        return attention_segment(p, line, blockIdx.x, pos, stop);
    }();
    if constexpr (PAGED) ended = seg;
    const AttentionItem& it = seg.it;
    if (!it.live) break;
    const AttentionRow row = attention_row(p, it, fr);
    const int key_head = attention_key_head(p, it.head_block);
    const int last_token = min(it.seq.nq, (it.tile + 1) * p.tile_tokens) - 1;
    const int tile_limit = attention_limit(p, it.seq, last_token);
    const int first = (int)min((uint64_t)seg.first << line.unit_shift, (uint64_t)INT32_MAX);
    const int last = (int)min((uint64_t)tile_limit, (uint64_t)(seg.first + seg.count) << line.unit_shift);
    const int limit = row.live ? min(attention_limit(p, it.seq, row.token), last) : last;
    // Keys that every row sees.
    const int open = min(attention_limit(p, it.seq, min(it.tile * p.tile_tokens, it.seq.nq)), last);

    const int drow = lane / L::CHUNKS, dslot = lane % L::CHUNKS;
    const uint8_t *kb = nullptr, *vb = nullptr;  // rows: of this sequence and key head
    uint32_t kts = 0, vts = 0;
    if constexpr (!PAGED) {
      kb = reinterpret_cast<const uint8_t*>(p.k + (int64_t)it.seq.k0 * p.k_ts + (int64_t)key_head * p.k_hs);
      vb = reinterpret_cast<const uint8_t*>(p.v + (int64_t)it.seq.k0 * p.v_ts + (int64_t)key_head * p.v_hs);
      kts = (uint32_t)p.k_ts * 2;
      vts = (uint32_t)p.v_ts * 2;
    }
    struct Halves {
      int64_t page[2];
    };
    // The pages of a block's halves, by scalar loads that are waited for where they are used.
    auto look = [&](int key0) {
      Halves h{{-1, -1}};
      if constexpr (PAGED) {
        if (last > 0) {
          typedef const __attribute__((address_space(4))) int64_t table_t;
          table_t* row = (table_t*)(uintptr_t)(p.cache.table + (int64_t)it.seq.k0 * p.cache.width);
          static_for<2>([&](auto i) { h.page[i] = row[min(key0 + 16 * i, last - 1) >> p.cache.page_shift]; });
        }
      }
      return h;
    };
    auto issue = [&](int buf, int key0, const Halves& halves) {
      const int left = last - key0;  // none: every lane reads zeros
      const uint32_t dst = ring_lds + buf * L::SLOT;
      if constexpr (!PAGED) {
        const __amdgpu_buffer_rsrc_t rk = make_rsrc(kb + (int64_t)key0 * kts, 0x7fffffffu);
        const __amdgpu_buffer_rsrc_t rv = make_rsrc(vb + (int64_t)key0 * vts, 0x7fffffffu);
        static_for<L::TILE / 1024>([&](auto i) {
          const int r = drow + i * L::ROWS;
          const int c = dslot ^ step_k_swizzle<L::PITCH>(r);
          lds_dma16(rk, dst + i * 1024, r < left && c * 8 < p.dim ? (uint32_t)r * kts + c * 16 : VFA_OOB);
        });
        static_for<L::TILE / 1024>([&](auto i) {
          const int r = drow + i * L::ROWS;
          const int c = dslot ^ step_v_swizzle<L::PITCH>(r);
          lds_dma16(rv, dst + L::TILE + i * 1024, r < left && c * 8 < p.dim ? (uint32_t)r * vts + c * 16 : VFA_OOB);
        });
      } else {
        constexpr int PER = L::TILE / 2048;  // instructions of 16 keys
        const uint32_t row_bytes = (uint32_t)p.dim * (E4M3 ? 1 : 2);
        const int64_t head_rows = (int64_t)p.cache.key_heads << p.cache.page_shift;  // from a page's keys to its values
        static_for<2>([&](auto h) {
          const int64_t page = halves.page[h];
          const bool none = (uint64_t)page >= (uint64_t)p.cache.pages;  // reads zeros
          const uint32_t size = none ? 0 : 0x7fffffffu;
          const int64_t row = none ? 0
                                   : 2 * page * head_rows + ((int64_t)key_head << p.cache.page_shift) +
                                         ((key0 + 16 * h) & ((1 << p.cache.page_shift) - 1));
          const uint8_t* at = p.cache.values + row * row_bytes;
          const __amdgpu_buffer_rsrc_t rk = make_rsrc(at, size), rv = make_rsrc(at + head_rows * row_bytes, size);
          static_for<PER>([&](auto i) {
            const int r = drow + (h * PER + i) * L::ROWS;
            const int c = dslot ^ (E4M3 ? step_k_code_swizzle<L::PITCH>(r) : step_k_swizzle<L::PITCH>(r));
            lds_dma16(rk, dst + (h * PER + i) * 1024,
                      r < left && (uint32_t)c * 16 < row_bytes ? (uint32_t)(r - 16 * h) * row_bytes + c * 16 : VFA_OOB);
          });
          static_for<PER>([&](auto i) {
            const int r = drow + (h * PER + i) * L::ROWS;
            const int c = dslot ^ (E4M3 ? step_v_code_swizzle<L::PITCH>(r) : step_v_swizzle<L::PITCH>(r));
            lds_dma16(rv, dst + L::TILE + (h * PER + i) * 1024,
                      r < left && (uint32_t)c * 16 < row_bytes ? (uint32_t)(r - 16 * h) * row_bytes + c * 16 : VFA_OOB);
          });
          if constexpr (E4M3)  // 16 keys' factors, then 16 values'
            lds_dma4(make_rsrc(p.cache.scales + row, size), dst + 2 * L::TILE + h * 256,
                     lane < 32 && 16 * h + (lane & 15) < left
                         ? 4 * ((uint32_t)(lane & 15) + (lane & 16 ? (uint32_t)head_rows : 0)) : VFA_OOB);
        });
      }
    };
    constexpr int STRIDE = L::WAVES * L::KEYS;
    const int start = first + wave * L::KEYS;
    Halves next;
    {
      Halves begun[L::NS];
      static_for<L::NS>([&](auto i) { begun[i] = look(start + i * STRIDE); });
      static_for<L::NS>([&](auto i) { issue(i, start + i * STRIDE, begun[i]); });
      next = look(start + L::NS * STRIDE);
    }

    v4i q[QS];
    static_for<QS>([&](auto s) { q[s] = attention_query(p, it, row, s * 32 + fg * 8); });
    v4f o[DB];
    static_for<DB>([&](auto i) { o[i] = v4f{}; });
    float m = VFA_LOWEST, l = 0;
    bool far = false;
    const uint8_t* krow = ring + fr * L::PITCH + (E4M3 ? (fg & 1) * 8 : 0);
    const int ksw = E4M3 ? step_k_code_swizzle<L::PITCH>(fr) : step_k_swizzle<L::PITCH>(fr);
    const int vr = E4M3 ? 4 * fg + (lane >> 1 & 3) + (lane & 8) * 2 : 4 * fg + ((lane >> 2) & 3);
    const int vc = (lane & 3) >> 1;
    const uint8_t* vrow = ring + L::TILE + vr * L::PITCH + (lane & 1) * 8;
    const int vsw = E4M3 ? step_v_code_swizzle<L::PITCH>(vr) : step_v_swizzle<L::PITCH>(vr);
    const uint8_t* factors = ring + 2 * L::TILE + 16 * fg;

    int buf = 0;
    for (int key0 = start; key0 < last; key0 += STRIDE, buf = buf + 1 == L::NS ? 0 : buf + 1) {
      wait_vmcnt<(L::NS - 1) * L::DMA, false>();
      asm volatile("" ::: "memory");
      v4f s[2];
      static_for<2>([&](auto kbk) {
        s[kbk] = v4f{};
        static_for<QS>([&](auto st) {
          const uint8_t* src = krow + buf * L::SLOT + kbk * 16 * L::PITCH;
          v4i a;
          if constexpr (E4M3) a = attention_widen<F16>(*reinterpret_cast<const v2i*>(src + (((2 * st + (fg >> 1)) ^ ksw) << 4)));
          else a = *reinterpret_cast<const v4i*>(src + (((4 * st + fg) ^ ksw) << 4));
          s[kbk] = mfma16<F16>(a, q[st], s[kbk]);
        });
        if constexpr (E4M3) s[kbk] *= *reinterpret_cast<const v4f*>(factors + buf * L::SLOT + kbk * 256);
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
      const float ref = attention_shift<W16>(p) - attention_top(m, p.c);
      v4i pk;
      [[maybe_unused]] v4i rest;
      auto weights = [&](auto far_rows) {
        static_for<4>([&](auto j) {
          constexpr int r = (j % 2) * 2;
          const float w0 = attention_weight<far_rows>(s[j / 2][r], p.c, m, ref, attention_shift<W16>(p));
          const float w1 = attention_weight<far_rows>(s[j / 2][r + 1], p.c, m, ref, attention_shift<W16>(p));
          if constexpr (E4M3) {
            const v2f f = *reinterpret_cast<const v2f*>(factors + buf * L::SLOT + (j / 2) * 256 + 64 + r * 4);
            pk[(int)j] = pack2<W16>(w0 * f[0], w1 * f[1]);
            if constexpr (F16) rest[(int)j] = attention_rest(w0 * f[0], w1 * f[1], pk[(int)j]);
            l += w0 + w1;
          } else {
            pk[(int)j] = pack2<W16>(w0, w1);
            l = attention_sum2<W16>(pk[(int)j], l);
          }
        });
      };
      if (far) weights(std::true_type{});
      else weights(std::false_type{});
      static_for<DB>([&](auto db) {
        if constexpr (E4M3) {
          const v4i a = attention_widen<false>(lds_read_tr8(vrow + buf * L::SLOT + ((db ^ vsw) << 4)));
          o[db] = mfma16<W16>(a, pk, o[db]);
          if constexpr (F16) o[db] = mfma16<W16>(a, rest, o[db]);
        } else {
          const uint8_t* src = vrow + buf * L::SLOT + (((2 * db + vc) ^ vsw) << 4);
          const v2i lo = lds_read_tr16(src), hi = lds_read_tr16(src + 16 * L::PITCH);
          o[db] = mfma16<W16>(v4i{lo[0], lo[1], hi[0], hi[1]}, pk, o[db]);
        }
      });
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot is read
      asm volatile("" ::: "memory");
      issue(buf, key0 + L::NS * STRIDE, next);
      next = look(key0 + (L::NS + 1) * STRIDE);
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
    // Thread t: row t / 16 (and those 4 WAVES further), the d of t % 16 in runs of four.
    const int e = (int)threadIdx.x & 15;
#pragma unroll
    for (int turn = 0; turn < 4 / L::WAVES; ++turn) {
      const int r = ((int)threadIdx.x >> 4) + turn * (4 * L::WAVES);
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
    }
    pos += seg.count;
    if (pos < stop) __syncthreads();  // the sums are read: the rings may be filled again
  }
  if constexpr (PAGED) {
    if (p.begun && threadIdx.x == 0) {
      const AttentionBegun own = attention_begun(p, line, blockIdx.x, ended, stop);
      *reinterpret_cast<v4i*>(p.begun + 4 * blockIdx.x) = v4i{own.segments, own.row, own.tokens, own.head_block};
    }
  }
}

// The sum over a tile's segments: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  Workgroup b
// takes the tile that workgroup b of attention_step began and did not end.  Thread t: d 4 (t % 16) and
// 64 more, one row, every groups-th segment under a maximum of its own; the groups meet in LDS.
template <bool F16, bool PAGED, int THREADS>
__global__ void __launch_bounds__(THREADS) attention_step_join(const AttentionParams p) {
  AttentionItem it{};
  int segments;
  if constexpr (PAGED) {
    const v4i begun = *reinterpret_cast<const v4i*>(p.begun + 4 * blockIdx.x);
    auto u = [&](int i) { return __builtin_amdgcn_readfirstlane(begun[i]); };
    segments = u(0);
    if (segments == 0) return;
    it.seq = AttentionSeq{u(1), 0, u(2), 0};
    it.head_block = u(3);
  } else {
    const AttentionLine line = attention_line(p, gridDim.x);
    const int part = blockIdx.x >> (line.xcds == 8 ? 3 : 0);
    const uint32_t begin = part * line.quota, stop = min(begin + line.quota, line.end);
    if (begin >= stop) return;
    const AttentionSegment seg = attention_segment(p, line, blockIdx.x, stop - 1, line.end);
    const uint32_t tile_begin = stop - 1 - seg.first, tile_end = tile_begin + seg.of;
    if (!seg.it.live || tile_begin < begin || tile_end <= stop) return;
    segments = (int)((tile_end - 1) / line.quota) - part + 1;
    it = seg.it;
  }
  // Segment s lies in workgroup blockIdx.x + xcds s, slot 1 for the first, 0 for the others.
  const int xcds = p.head_blocks % 8 == 0 ? 8 : 1;
  auto slot = [&](int s) { return 2 * ((int64_t)blockIdx.x + xcds * s) + (s == 0); };
  const int tokens = min(p.tile_tokens, it.seq.nq - it.tile * p.tile_tokens);
  const int rows = min(16, tokens * p.heads_per_tile);
  const int pow = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  const int groups = min(16, THREADS / 16 / pow);
  const int e = (int)threadIdx.x & 15, r = (int)threadIdx.x / 16 % pow, sg = (int)threadIdx.x / 16 / pow;
  __shared__ float sums[THREADS / 16][132];
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
  const AttentionRow row = attention_row(p, it, r);
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
  uint16_t* dst = p.out + (int64_t)(it.seq.q0 + row.token) * p.o_ts + (int64_t)row.head * p.o_hs;
  static_for<2>([&](auto h) {
    const int d = 4 * e + 64 * h;
    const v4f y = l == 0 ? v4f{} : x[h] * inv;
    if (d < p.dim) *reinterpret_cast<v2i*>(dst + d) = v2i{pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3])};
  });
}

template <bool F16, int STORE, int W>
static void launch_step(const AttentionParams& p, int grid, int join, hipStream_t s) {
  const dim3 g((unsigned)grid), b(64 * W);
  if (p.dim <= 64) attention_step<F16, 64, STORE, W><<<g, b, 0, s>>>(p);
  else attention_step<F16, 128, STORE, W><<<g, b, 0, s>>>(p);
  if (join == 1) attention_step_join<F16, STORE != kStoreRows, 1024><<<g, dim3(1024), 0, s>>>(p);
  if constexpr (STORE != kStoreRows)
    if (join == 2) attention_step_join<F16, true, 256><<<g, dim3(256), 0, s>>>(p);
}

void launch_attention_step(const AttentionParams& p, bool f16, AttentionStore store, int grid, int waves, int join,
                           hipStream_t s) {
  auto of = [&](auto stored, auto w) {
    if (f16) launch_step<true, stored, w>(p, grid, join, s);
    else launch_step<false, stored, w>(p, grid, join, s);
  };
  auto paged = [&](auto stored) {
    if (waves == 1) of(stored, std::integral_constant<int, 1>{});
    else if (waves == 2) of(stored, std::integral_constant<int, 2>{});
    else of(stored, std::integral_constant<int, 4>{});
  };
  if (store == kStoreE4M3) paged(std::integral_constant<int, kStoreE4M3>{});
  else if (store == kStorePages) paged(std::integral_constant<int, kStorePages>{});
  else of(std::integral_constant<int, kStoreRows>{}, std::integral_constant<int, 4>{});
}

}  // namespace vfa
