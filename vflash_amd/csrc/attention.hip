// Packed attention for gfx950: tiles of many rows, and the sum over split keys.
//
// The scores are computed transposed, S^T = K Q^T, with v_mfma_f32_32x32x16: a lane then holds
// 16 keys of one row of the tile per block of 32 keys, so that the row's running maximum m, its
// sum and its mask limit are one register each, the softmax needs one exchange between the half
// waves, and the values p are the second product's operand as they lie: O^T = V^T P^T with K
// position (half h, j) of a step of 16 keys standing for key 4 h + j (j < 4) or 8 + 4 h + j - 4.
// V^T is read from the row-major tile by transposing LDS reads, four keys at a time.
//
// A workgroup's waves, 32 rows each, share tiles of 64 keys in LDS, which DMA fills one tile
// ahead.  Weights are rounded to the operands' type, as the matrix instruction takes them (by half a
// step at most, 2^-8 of the value in bf16 and 2^-11 in f16), and the binary32 sum that normalises them
// is that of the rounded ones: errors against 64 bits are 1.1 to 1.4 times those of weights in 32 bits.
//
// Bound by the softmax beside the MFMAs, and over milliseconds by the board's power: 32760 tokens
// of 40 heads of 128, unmasked, 19.8 ms (1.11 PFLOP/s, MFMAs busy 0.60 of the cycles at 1.65 GHz, VALU
// 0.50); 8191 causal tokens of 16 heads of 64 0.165 ms (0.83 PFLOP/s; VALU 0.54, MFMAs 0.38: a wave's
// products and softmax follow each other, and the others' fill its gaps in part); 24 causal prompts of
// up to 1023 tokens, 28 heads over 4, 0.126 ms (VALU 0.43, MFMAs 0.30).  Cards differ by 5 %.  Blocks of
// 32 keys above dimension 64 let three workgroups share a CU, 64 below four.
//
// A paged cache differs in where a wave's part of a tile comes from: rows of one 16 keys, which lie in one page.
// E4M3 codes go through registers, a tile ahead, and reach LDS as 16-bit numbers (exactly), converted once for
// all waves; a key's factor multiplies its score, a value's its weight before that is rounded, to bf16
// (for f16 queries to two of it).
#include "attention_codes.h"
#include "attention_plan.h"

namespace vfa {

template <int DP>
struct AttentionTiles {
  static constexpr int PITCH = DP <= 64 ? 128 : 256, CHUNKS = PITCH / 16, ROWS = 1024 / PITCH;
  static constexpr int KEYS = DP <= 64 ? 64 : 32, KB = KEYS / 32, TILE = KEYS * PITCH, SLOT = 2 * TILE;
};
// The 16-byte chunk c of row r lies in slot c ^ key.  K: the 16 rows of a ds_read_b128 phase take
// different slots.  V: the four rows x four chunks that a half wave's transposing read takes do.
template <int PITCH>
__device__ __forceinline__ int k_swizzle(int r) {
  return PITCH == 256 ? r & 15 : lds_swizzle(r);
}
template <int PITCH>
__device__ __forceinline__ int v_swizzle(int r) {
  return PITCH == 256 ? (r & 3) << 2 : (r >> 1 & 1) << 2;
}

template <bool F16, int DP, int WAVES, int STORE>
__global__ void __launch_bounds__(64 * WAVES, (DP <= 64 ? 4 : 3) - (STORE == kStoreE4M3)) attention_tiles(const AttentionParams p) {
  using L = AttentionTiles<DP>;
  constexpr bool PAGED = STORE != kStoreRows, E4M3 = STORE == kStoreE4M3;
  constexpr bool W16 = F16 && !E4M3;  // the type of the weights
  constexpr int QS = DP / 16, DB = DP / 32;            // contraction steps, blocks of 32 d
  constexpr int BLOCKS = L::TILE / 1024 / WAVES;       // DMA instructions per wave for K, and for V
  static_assert(L::TILE % (1024 * WAVES) == 0, "DMA blocks");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * L::SLOT];
  __shared__ float factors[E4M3 ? 2 : 1][2][E4M3 ? L::KEYS : 1];  // of keys and values
  const AttentionItem it = attention_item<false, PAGED>(p, blockIdx.x);
  if (!it.live) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = (int)threadIdx.x & 63;
  const int fr = lane & 31, fh = lane >> 5;
  const uint32_t base_lds = __builtin_amdgcn_readfirstlane(lds_addr(lds));

  const AttentionRow row = attention_row(p, it, wave * 32 + fr);
  const int part_head = attention_key_head(p, it.head_block);
  // Keys of this item: [first, last), last no further than the tile's last token sees.
  const int last_token = min(it.seq.nq, (it.tile + 1) * p.tile_tokens) - 1;
  const int tile_limit = attention_limit(p, it.seq, last_token);
  const int first = it.split * it.chunk;
  const int last = (int)min((int64_t)tile_limit, (int64_t)first + it.chunk);
  const int limit = row.live ? attention_limit(p, it.seq, row.token) : last;
  // Of this wave: the keys before which no row masks anything, and after which all do.
  const int wave_first_token = min(it.tile * p.tile_tokens + attention_token_of(p, wave * 32), it.seq.nq);
  const int wave_last_token = min(it.tile * p.tile_tokens + min(attention_token_of(p, wave * 32 + 31), p.tile_tokens - 1),
                                  it.seq.nq - 1);
  const int open = min(attention_limit(p, it.seq, wave_first_token), last);
  const int end = min(attention_limit(p, it.seq, wave_last_token), last);

  const uint8_t *kb = nullptr, *vb = nullptr;  // rows: of this sequence and key head
  uint32_t kts = (uint32_t)p.dim * 2, vts = kts;  // bytes of a row
  if constexpr (!PAGED) {
    kb = reinterpret_cast<const uint8_t*>(p.k + (int64_t)it.seq.k0 * p.k_ts + (int64_t)part_head * p.k_hs);
    vb = reinterpret_cast<const uint8_t*>(p.v + (int64_t)it.seq.k0 * p.v_ts + (int64_t)part_head * p.v_hs);
    kts = (uint32_t)p.k_ts * 2;
    vts = (uint32_t)p.v_ts * 2;
  }
  // DMA: block i of this wave holds rows (wave * BLOCKS + i) * ROWS + lane / CHUNKS; lane l fills
  // slot l % CHUNKS.  Rows past the keys and chunks past the head read as zeros.
  constexpr int WAVE_ROWS = BLOCKS * L::ROWS;
  static_assert(16 % WAVE_ROWS == 0, "a wave's rows lie in one page");
  const int drow = wave * WAVE_ROWS + lane / L::CHUNKS, dslot = lane % L::CHUNKS;
  // Pages: the 16 keys that this wave's rows are some of.
  const int group = wave * WAVE_ROWS / 16 * 16;
  const int64_t head_rows = (int64_t)p.cache.key_heads << p.cache.page_shift;  // from a page's keys to its values
  auto look = [&](int key0) {  // a scalar load, waited for where it is used
    if constexpr (PAGED) {
      typedef const __attribute__((address_space(4))) int64_t table_t;
      if (key0 + group < last)
        return (int64_t)((table_t*)(uintptr_t)(p.cache.table + (int64_t)it.seq.k0 * p.cache.width))[(key0 + group) >> p.cache.page_shift];
    }
    return (int64_t)-1;
  };
  // The cache's row of key `key` on `page`, as keys count.
  auto cache_row = [&](int64_t page, int key) {
    return 2 * page * head_rows + ((int64_t)part_head << p.cache.page_shift) + (key & ((1 << p.cache.page_shift) - 1));
  };
  auto issue = [&](int buf, int key0, int64_t page) {
    const int left = last - key0;
    const uint32_t dst = base_lds + buf * L::SLOT + wave * BLOCKS * 1024;
    const uint32_t from = PAGED ? (uint32_t)group : 0;  // the first row of the resources
    __amdgpu_buffer_rsrc_t rk, rv;
    if constexpr (PAGED) {
      const bool none = (uint64_t)page >= (uint64_t)p.cache.pages;  // reads zeros
      const uint8_t* at = p.cache.values + (none ? 0 : cache_row(page, key0 + group) * p.dim * 2);
      rk = make_rsrc(at, none ? 0 : 0x7fffffffu);
      rv = make_rsrc(at + head_rows * p.dim * 2, none ? 0 : 0x7fffffffu);
    } else {
      rk = make_rsrc(kb + (int64_t)key0 * kts, 0x7fffffffu);
      rv = make_rsrc(vb + (int64_t)key0 * vts, 0x7fffffffu);
    }
    static_for<BLOCKS>([&](auto i) {
      const int r = drow + i * L::ROWS;
      const int c = dslot ^ k_swizzle<L::PITCH>(r);
      const uint32_t off = ((uint32_t)r - from) * kts + c * 16;
      lds_dma16(rk, dst + i * 1024, r < left && c * 8 < p.dim ? off : VFA_OOB);
    });
    static_for<BLOCKS>([&](auto i) {
      const int r = drow + i * L::ROWS;
      const int c = dslot ^ v_swizzle<L::PITCH>(r);
      const uint32_t off = ((uint32_t)r - from) * vts + c * 16;
      lds_dma16(rv, dst + L::TILE + i * 1024, r < left && c * 8 < p.dim ? off : VFA_OOB);
    });
  };
  // E4M3: thread t takes 16 codes of a key and of its value, one of the first threads also a factor.
  constexpr int CODE_CHUNKS = L::CHUNKS / 2;
  static_assert(!E4M3 || L::KEYS * CODE_CHUNKS == 64 * WAVES, "a chunk a thread");
  const int crow = (int)threadIdx.x / CODE_CHUNKS, cchunk = (int)threadIdx.x % CODE_CHUNKS;
  v4i key_codes, value_codes;
  float factor;
  auto fetch = [&](int key0, int64_t page) {
    key_codes = value_codes = v4i{};
    factor = 0;
    if ((uint64_t)page < (uint64_t)p.cache.pages && key0 + crow < last && cchunk * 16 < p.dim) {
      const uint8_t* at = p.cache.values + cache_row(page, key0 + crow) * p.dim + cchunk * 16;
      key_codes = *reinterpret_cast<const v4i*>(at);
      value_codes = *reinterpret_cast<const v4i*>(at + head_rows * p.dim);
    }
    const int t = (int)threadIdx.x, key = key0 + t % L::KEYS;
    if (t < 2 * L::KEYS && key < last) {
      const int64_t own = p.cache.table[(int64_t)it.seq.k0 * p.cache.width + (key >> p.cache.page_shift)];
      if ((uint64_t)own < (uint64_t)p.cache.pages) factor = p.cache.scales[cache_row(own, key) + (t < L::KEYS ? 0 : head_rows)];
    }
  };
  auto place = [&](int buf) {
    uint8_t* at = lds + buf * L::SLOT + crow * L::PITCH;
    static_for<2>([&](auto h) {
      const int c = 2 * cchunk + h;
      *reinterpret_cast<v4i*>(at + ((c ^ k_swizzle<L::PITCH>(crow)) << 4)) = attention_widen<F16>(v2i{key_codes[2 * h], key_codes[2 * h + 1]});
      *reinterpret_cast<v4i*>(at + L::TILE + ((c ^ v_swizzle<L::PITCH>(crow)) << 4)) =
          attention_widen<false>(v2i{value_codes[2 * h], value_codes[2 * h + 1]});
    });
    const int t = (int)threadIdx.x;
    if (t < 2 * L::KEYS) factors[buf][t / L::KEYS][t % L::KEYS] = factor;
  };

  int64_t next = -1;  // the page of the tile after the one on its way
  if (first < last) {
    if constexpr (E4M3) fetch(first, look(first));
    else issue(0, first, look(first));
    next = look(first + L::KEYS);
  }
  v4i q[QS];
  static_for<QS>([&](auto s) { q[s] = attention_query(p, it, row, s * 16 + fh * 8); });
  v16f o[DB];
  static_for<DB>([&](auto i) { o[i] = v16f{}; });
  float m = VFA_LOWEST, l = 0;
  bool far = false;

  // LDS addresses of this lane's fragments.
  const uint8_t* krow = lds + fr * L::PITCH;
  const int ksw = k_swizzle<L::PITCH>(fr);
  // Transposing reads: lane 4 r + c of a group of 16 gives row r, elements 4 c; the group covers
  // d 16 (group % 2) .. + 15 of a block, the half wave's rows start at 4 fh.
  const int vr = 4 * fh + ((lane >> 2) & 3);
  const int vc = (lane >> 4 & 1) * 2 + ((lane & 3) >> 1);
  const uint8_t* vrow = lds + L::TILE + vr * L::PITCH + (lane & 1) * 8;
  const int vsw = v_swizzle<L::PITCH>(vr);  // rows 8 apart share it

  if constexpr (E4M3) {
    if (first < last) place(0);
    __syncthreads();
  }
  for (int key0 = first, buf = 0; key0 < last; key0 += L::KEYS, buf ^= 1) {
    const bool more = key0 + L::KEYS < last;
    if constexpr (E4M3) {
      // This tile's other buffer is written at the end, after the barrier of the one before.
      if (more) {
        fetch(key0 + L::KEYS, next);
        next = look(key0 + 2 * L::KEYS);
      }
    } else {
      wait_vmcnt<0, false>();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();  // this tile has landed for every wave, and the other buffer is read
      asm volatile("" ::: "memory");
      if (more) {
        issue(buf ^ 1, key0 + L::KEYS, next);
        next = look(key0 + 2 * L::KEYS);
      }
    }
    auto after = [&] {
      if constexpr (E4M3) {
        if (more) place(buf ^ 1);
        __syncthreads();
      }
    };
    if (key0 >= end) {
      after();
      continue;
    }
    v16f s[L::KB];
    static_for<L::KB>([&](auto kbk) { s[kbk] = v16f{}; });
    static_for<QS>([&](auto st) {
      static_for<L::KB>([&](auto kbk) {
        const v4i a = *reinterpret_cast<const v4i*>(krow + buf * L::SLOT + kbk * 32 * L::PITCH +
                                                    (((2 * st + fh) ^ ksw) << 4));
        s[kbk] = mfma32<F16>(a, q[st], s[kbk]);
      });
    });
    if constexpr (E4M3)
      static_for<4 * L::KB>([&](auto g) {
        const v4f f = *reinterpret_cast<const v4f*>(&factors[buf][0][8 * g + 4 * fh]);
        static_for<4>([&](auto r) { s[g / 4][(int)(g % 4 * 4 + r)] *= f[(int)r]; });
      });
    if (key0 + L::KEYS > open) {  // some row of the wave masks some key
      const int lim = limit - key0 - 4 * fh;
      static_for<L::KB>([&](auto kbk) {
        static_for<16>([&](auto r) {
          const int key = kbk * 32 + 8 * (r / 4) + r % 4;
          s[kbk][(int)r] = key < lim ? s[kbk][(int)r] : -__builtin_inff();
        });
      });
    }
    v4i pk[2 * L::KB];
    [[maybe_unused]] v4i rest[E4M3 && F16 ? 2 * L::KB : 1];
    float sum;
    auto weights = [&](auto far_rows) {
      const float ref = attention_shift<W16>(p) - attention_top(m, p.c);
      sum = 0;
      static_for<2 * L::KB>([&](auto st) {
        static_for<4>([&](auto j) {
          constexpr int r = (st % 2) * 8 + 2 * j;
          const float w0 = attention_weight<far_rows>(s[st / 2][r], p.c, m, ref, attention_shift<W16>(p));
          const float w1 = attention_weight<far_rows>(s[st / 2][r + 1], p.c, m, ref, attention_shift<W16>(p));
          if constexpr (E4M3) {
            const v2f f = *reinterpret_cast<const v2f*>(&factors[buf][1][st / 2 * 32 + 8 * (r / 4) + 4 * fh + r % 4]);
            pk[st][(int)j] = pack2<W16>(w0 * f[0], w1 * f[1]);
            if constexpr (F16) rest[st][(int)j] = attention_rest(w0 * f[0], w1 * f[1], pk[st][(int)j]);
            sum += w0 + w1;
          } else {
            pk[st][(int)j] = pack2<W16>(w0, w1);
            sum = attention_sum2<W16>(pk[st][(int)j], sum);
          }
        });
      });
    };
    if (far) weights(std::true_type{});
    else weights(std::false_type{});
    if (__builtin_amdgcn_ballot_w64(!(sum <= attention_bound<W16>(p)))) {
      // The first keys that a row sees, or scores far above those before.
      float mx = s[0][0];
      static_for<16 * L::KB - 1>([&](auto r) { mx = fmaxf(mx, s[(r + 1) / 16][(int)((r + 1) % 16)]); });
      const float next = fmaxf(m, max_across32(mx)), f = __builtin_amdgcn_exp2f((m - next) * p.c);
      static_for<DB>([&](auto i) { static_for<16>([&](auto r) { o[i][(int)r] *= f; }); });
      l *= f;
      m = next;
      far = __builtin_amdgcn_ballot_w64(fabsf(m * p.c) >= kAttentionFar && m > VFA_LOWEST) != 0;
      if (far) weights(std::true_type{});
      else weights(std::false_type{});
    }
    l += sum;
    static_for<2 * L::KB>([&](auto st) {
      static_for<DB>([&](auto db) {
        const uint8_t* src = vrow + buf * L::SLOT + st * 16 * L::PITCH + (((4 * db + vc) ^ vsw) << 4);
        const v2i lo = lds_read_tr16(src), hi = lds_read_tr16(src + 8 * L::PITCH);
        o[db] = mfma32<W16>(v4i{lo[0], lo[1], hi[0], hi[1]}, pk[st], o[db]);
        if constexpr (E4M3 && F16) o[db] = mfma32<W16>(v4i{lo[0], lo[1], hi[0], hi[1]}, rest[st], o[db]);
      });
    });
    after();
  }
  l = sum_across32(l);

  if (it.splits > 1) {
    if (first >= tile_limit) return;  // attention_join does not read it
    const int64_t at = (int64_t)(it.slot + it.split) * (32 * WAVES) + wave * 32 + fr;
    float* dst = p.part + at * p.dim;
    static_for<DB>([&](auto db) {
      static_for<4>([&](auto r4) {
        const int d = db * 32 + r4 * 8 + fh * 4;
        if (d < p.dim)
          *reinterpret_cast<v4f*>(dst + d) = v4f{o[db][r4 * 4], o[db][r4 * 4 + 1], o[db][r4 * 4 + 2], o[db][r4 * 4 + 3]};
      });
    });
    if (fh == 0) *reinterpret_cast<v2f*>(p.part_ml + at * 2) = v2f{attention_top(m, p.c), l};
    return;
  }
  const bool none = l == 0;  // the row sees nothing
  const float inv = 1.0f / l;
  uint16_t* dst = p.out + (int64_t)(it.seq.q0 + row.token) * p.o_ts + (int64_t)row.head * p.o_hs;
  static_for<DB>([&](auto db) {
    static_for<2>([&](auto r8) {
      // Two runs of four d, eight apart, become eight d in a row by one exchange of half waves.
      int w[4];
      static_for<2>([&](auto j) {
        auto at = [&](int r) { return none ? 0.0f : o[db][r] * inv; };
        const int a = pack2<F16>(at(r8 * 8 + 2 * j), at(r8 * 8 + 2 * j + 1));
        const int b = pack2<F16>(at(r8 * 8 + 4 + 2 * j), at(r8 * 8 + 4 + 2 * j + 1));
        const auto x = __builtin_amdgcn_permlane32_swap((uint32_t)a, (uint32_t)b, false, false);
        w[j] = (int)x[0];
        w[2 + j] = (int)x[1];
      });
      const int d = db * 32 + r8 * 16 + fh * 8;
      if (row.live && d < p.dim) *reinterpret_cast<v4i*>(dst + d) = v4i{w[0], w[1], w[2], w[3]};
    });
  });
}

// The sum over a tile's splits: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  A workgroup
// takes every eighth row of a tile, half a wave a row, four d a lane.
template <bool F16, bool PAGED>
__global__ void __launch_bounds__(256) attention_join(const AttentionParams p, int rows) {
  const AttentionItem it = attention_item<true, PAGED>(p, blockIdx.x);
  if (!it.live || it.splits == 1) return;
  const int d = 4 * ((int)threadIdx.x & 31);
  const int last_token = min(it.seq.nq, (it.tile + 1) * p.tile_tokens) - 1;
  const int tile_limit = attention_limit(p, it.seq, last_token);
  const int splits = (int)(((uint32_t)tile_limit + (uint32_t)it.chunk - 1) / (uint32_t)it.chunk);
#pragma unroll 2
  for (int r = blockIdx.y * 8 + ((int)threadIdx.x >> 5); r < rows; r += 8 * gridDim.y) {
    const AttentionRow row = attention_row(p, it, r);
    float top = VFA_LOWEST, l = 0;
    v4f x = v4f{};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const int64_t at = (int64_t)(it.slot + s) * rows + r;
      const v2f ml = *reinterpret_cast<const v2f*>(p.part_ml + at * 2);
      const v4f y = d < p.dim ? *reinterpret_cast<const v4f*>(p.part + at * p.dim + d) : v4f{};
      const float next = fmaxf(top, ml[0]);
      const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(ml[0] - next);
      top = next;
      l = l * old + f * ml[1];
      x = x * old + y * f;
    }
    x = l == 0 ? v4f{} : x * (1.0f / l);
    if (row.live && d < p.dim)
      *reinterpret_cast<v2i*>(p.out + (int64_t)(it.seq.q0 + row.token) * p.o_ts + (int64_t)row.head * p.o_hs + d) =
          v2i{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3])};
  }
}

// ---------------------------------------------------------------------------
void launch_attention_step(const AttentionParams&, bool, AttentionStore, int, int, int, hipStream_t);

namespace {

template <bool F16, int STORE>
void launch_tiles(const AttentionParams& p, const AttentionPlan& plan, hipStream_t s) {
  const dim3 g((unsigned)plan.grid), b(64 * kTileWaves);
  if (p.dim <= 32) attention_tiles<F16, 32, kTileWaves, STORE><<<g, b, 0, s>>>(p);
  else if (p.dim <= 64) attention_tiles<F16, 64, kTileWaves, STORE><<<g, b, 0, s>>>(p);
  else if (p.dim <= 96) attention_tiles<F16, 96, kTileWaves, STORE><<<g, b, 0, s>>>(p);
  else attention_tiles<F16, 128, kTileWaves, STORE><<<g, b, 0, s>>>(p);
  if (!plan.join) return;
  attention_join<F16, STORE != kStoreRows><<<dim3((unsigned)plan.join, 8), dim3(256), 0, s>>>(p, plan.rows);
}

int64_t workspace_of(const AttentionParams& p, const AttentionPlan& plan) { return p.slots * plan.rows * (p.dim + 2) * 4; }

bool plan_fits(const AttentionPlan& plan) {
  return plan.grid < (int64_t(1) << 24) && plan.join < (int64_t(1) << 24) &&
         plan.line < (int64_t(1) << 32) - (int64_t(1) << 24);
}

// The weights' range and the workspace's parts.  `above`: how far above 2^shift a weight may be, as a power of two.
void attention_memory(AttentionParams& p, const AttentionPlan& plan, int above, void* workspace) {
  int log = 0;  // at most 2^log keys
  while ((int64_t(1) << log) < p.keys) ++log;
  p.shift = -(float)(above + 1 + log);
  p.bound = exp2f((float)above + p.shift);
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + p.slots * plan.rows * p.dim;
}

}  // namespace

// Bytes of workspace that the call may use: partial sums of the splits.
int64_t attention_workspace(const AttentionParams& params) {
  AttentionParams p = params;
  const AttentionPlan plan = attention_plan(p);
  return workspace_of(p, plan);
}

int64_t paged_attention_workspace(const AttentionParams& params, bool e4m3) {
  AttentionParams p = params;
  const AttentionPlan plan = paged_attention_plan(p, e4m3);
  return workspace_of(p, plan) + (plan.step && plan.join ? 16 * plan.grid : 0);
}

// false: the grid would pass HIP's limit, or a line of attention_step 2^32 units (its workgroups'
// parts end at most a grid past the line).
bool attention_fits(const AttentionParams& params) {
  AttentionParams p = params;
  return plan_fits(attention_plan(p));
}

bool paged_attention_fits(const AttentionParams& params, bool e4m3) {
  AttentionParams p = params;
  return plan_fits(paged_attention_plan(p, e4m3));
}

hipError_t launch_attention(const AttentionParams& params, bool f16, void* workspace, hipStream_t s) {
  AttentionParams p = params;
  const AttentionPlan plan = attention_plan(p);
  attention_memory(p, plan, 20, workspace);
  if (plan.step) {
    launch_attention_step(p, f16, kStoreRows, (int)plan.grid, 4, (int)plan.join, s);
    return hipGetLastError();
  }
  if (f16) launch_tiles<true, kStoreRows>(p, plan, s);
  else launch_tiles<false, kStoreRows>(p, plan, s);
  return hipGetLastError();
}

hipError_t launch_paged_attention(const AttentionParams& params, bool f16, void* workspace, hipStream_t s) {
  AttentionParams p = params;
  const AttentionPlan plan = paged_attention_plan(p, p.cache.scales != nullptr);
  // The maximum is followed once it is 2^8 above: no shift for more, so that weights times the factors of small E4M3
  // values stay above bf16's subnormals.
  attention_memory(p, plan, (int)kAttentionSlack, workspace);
  const bool codes = p.cache.scales != nullptr;
  if (plan.step && plan.join) p.begun = reinterpret_cast<int32_t*>(p.part_ml + p.slots * plan.rows * 2);
  if (plan.step) {
    launch_attention_step(p, f16, codes ? kStoreE4M3 : kStorePages, (int)plan.grid, plan.waves, (int)plan.join, s);
    return hipGetLastError();
  }
  if (codes) {
    if (f16) launch_tiles<true, kStoreE4M3>(p, plan, s);
    else launch_tiles<false, kStoreE4M3>(p, plan, s);
  } else {
    if (f16) launch_tiles<true, kStorePages>(p, plan, s);
    else launch_tiles<false, kStorePages>(p, plan, s);
  }
  return hipGetLastError();
}

}  // namespace vfa
