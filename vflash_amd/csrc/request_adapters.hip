// The low-rank adapters of many requests beside a shared projection, for gfx950:
//   out[m] = base[m] + scaling[i][b] (x[m] A_i^T) B_i^T,  i = index[m] (none outside [0, adapters): out[m] = base[m]),
// column n taking branch b's part of A_i (the branches of a merged projection).
//
// Rows are taken by adapter, whatever their order: an item is up to 16 (or 64) rows of one adapter, so each
// adapter in use is read about once.  Two products on the matrix cores, v_mfma_f32_16x16x32 with the
// adapter's rows as operand A and the items' rows as operand B:
//   request_down  t = x A^T, binary32.  K is split over the waves of a workgroup and, where there are few items, over
//                 workgroups, whose sums are added in their order by the reader: no atomics.
//   request_up    t times scaling, as two 16-bit numbers (high and low part: 16 bits of t or more enter the product),
//                 times B; base is added and the sum rounded once.
// Bound by launches for a few rows, by the adapters' bytes for a decoding batch, and by base and out for prompts.
#include "request_adapters.h"

#include <type_traits>

#include "common.h"

namespace vfa {

int compute_units();

namespace {

constexpr int RD_WAVES = 8;  // of request_down: parts of K
constexpr int RU_WAVES = 4;  // of request_up: column tiles

struct RequestItem {
  int adapter, count;  // adapter -1: none; count 0: no such item
  int row;             // this lane's row (by lane % 16, of the first block)
};

// Item `index` of at most 64 rows, found by the wave: the adapters by their first row, their rows in order.
__device__ __forceinline__ RequestItem request_find(const RequestAdapterParams& p, int index, int* rows) {
  const int lane = (int)threadIdx.x & 63;
  int mine = -2;  // no row
  if (lane < p.rows) {
    const int64_t i = p.index[lane];
    mine = (uint64_t)i < (uint64_t)p.adapters ? (int)i : -1;
  }
  uint64_t left = __builtin_amdgcn_ballot_w64(mine != -2);
  RequestItem it{-1, 0, 0};
  while (left) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t same = __builtin_amdgcn_ballot_w64(mine == a);
    const int count = __popcll(same), items = (count + p.item_rows - 1) / p.item_rows;
    if (index < items) {
      // Lane l of the adapter's rows goes to its place among them.
      const int place = __popcll(same & ((uint64_t(1) << lane) - 1)) - index * p.item_rows;
      if (mine == a && place >= 0 && place < p.item_rows) rows[place] = lane;
      it.adapter = a;
      it.count = min(p.item_rows, count - index * p.item_rows);
      return it;
    }
    index -= items;
    left &= ~same;
  }
  return it;
}

// Item `index`, its rows in `rows` (LDS of this workgroup).
__device__ __forceinline__ RequestItem request_item(const RequestAdapterParams& p, int index, int* rows) {
  RequestItem it;
  if (!p.order) {
    // Every wave finds the same and writes the same.
    it = request_find(p, index, rows);
  } else {
    it.adapter = p.list[3 * index];
    const int first = p.list[3 * index + 1];
    it.count = p.list[3 * index + 2];
    if ((int)threadIdx.x < it.count) rows[threadIdx.x] = p.order[first + threadIdx.x];
  }
  it.adapter = __builtin_amdgcn_readfirstlane(it.adapter);
  it.count = __builtin_amdgcn_readfirstlane(it.count);
  __syncthreads();
  return it;
}

template <bool F16>
__device__ __forceinline__ float widen(uint32_t w, int half) {
  if constexpr (F16) return (float)__builtin_bit_cast(v2hf, w)[half];
  else return half ? bf16_hi(w) : bf16_lo(w);
}
template <bool F16>
__device__ __forceinline__ int pack(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(int, v2hf{(_Float16)a, (_Float16)b});
  else return __builtin_bit_cast(int, v2bf{(__bf16)a, (__bf16)b});
}

}  // namespace

// Rows by adapter, those with none last, and the items.  One workgroup: a histogram, its prefix sums, and the rows
// to their places (within an adapter in any order: no row's result depends on it).
__global__ void __launch_bounds__(1024) request_groups(const RequestAdapterParams p) {
  extern __shared__ int counts[];  // [adapters + 1] rows, then places; [1024] sums
  __shared__ int row_sums[1024], item_sums[1024];
  const int bins = p.adapters + 1, t = (int)threadIdx.x;
  for (int b = t; b < bins; b += 1024) counts[b] = 0;
  __syncthreads();
  auto bin_of = [&](int64_t m) {
    const int64_t i = p.index[m];
    return (uint64_t)i < (uint64_t)p.adapters ? (int)i : p.adapters;
  };
  for (int64_t m = t; m < p.rows; m += 1024) atomicAdd(&counts[bin_of(m)], 1);
  __syncthreads();
  // Thread t's bins are next to each other.
  const int per = (bins + 1023) / 1024, b0 = min(t * per, bins), b1 = min(b0 + per, bins);
  auto items_of = [&](int c) { return (c + p.item_rows - 1) / p.item_rows; };
  int rows = 0, items = 0;
  for (int b = b0; b < b1; ++b) {
    rows += counts[b];
    items += items_of(counts[b]);
  }
  row_sums[t] = rows;
  item_sums[t] = items;
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    const int r = t >= o ? row_sums[t - o] : 0, i = t >= o ? item_sums[t - o] : 0;
    __syncthreads();
    row_sums[t] += r;
    item_sums[t] += i;
    __syncthreads();
  }
  int row = row_sums[t] - rows, item = item_sums[t] - items;
  for (int b = b0; b < b1; ++b) {
    const int c = counts[b];
    for (int first = 0; first < c; first += p.item_rows, ++item) {
      p.list[3 * item] = b < p.adapters ? b : -1;
      p.list[3 * item + 1] = row + first;
      p.list[3 * item + 2] = min(p.item_rows, c - first);
    }
    counts[b] = row;
    row += c;
  }
  for (int i = item_sums[1023] + t; i < p.items; i += 1024) p.list[3 * i + 2] = 0;
  __syncthreads();
  for (int64_t m = t; m < p.rows; m += 1024) p.order[atomicAdd(&counts[bin_of(m)], 1)] = (int)m;
}

// t of one item for RK blocks of 16 adapter rows and one split of K.
template <bool F16, int RB, int RK>
__global__ void __launch_bounds__(64 * RD_WAVES) request_down(const RequestAdapterParams p) {
  __shared__ int rows[RB * 16];
  __shared__ v4f part[RD_WAVES][RB * RK][64];
  const RequestItem it = request_item(p, (int)blockIdx.x, rows);
  if (it.count == 0 || it.adapter < 0) return;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int all = p.branches * p.width, r0 = (int)blockIdx.z * RK * 16;
  const int rank = p.ranks[it.adapter];

  // Blocks of adapter rows that hold some of the rank.
  bool used[RK], any = false;
  const uint16_t *xr[RB], *ar[RK];
  static_for<RK>([&](auto j) {
    const int r = r0 + j * 16;
    used[j] = r < all && r % p.width < rank;
    any = any || used[j];
    ar[j] = p.down + ((int64_t)it.adapter * all + min(r + fr, all - 1)) * p.k;
  });
  if (!any) return;
  static_for<RB>([&](auto i) { xr[i] = p.x + (int64_t)rows[min((int)i * 16 + fr, it.count - 1)] * p.ldx; });
  const int steps = (int)((p.k + 31) / 32);
  const int from = (int)blockIdx.y * p.steps, to = min(from + p.steps, steps);
  const int s0 = from + max(0, to - from) * wave / RD_WAVES, s1 = from + max(0, to - from) * (wave + 1) / RD_WAVES;

  constexpr int AHEAD = RB * RK >= 4 ? 2 : 4;
  v4f acc[RB][RK];
  static_for<RB>([&](auto i) { static_for<RK>([&](auto j) { acc[i][j] = v4f{}; }); });
  for (int s = s0; s < s1; s += AHEAD) {
    v4i xv[AHEAD][RB], av[AHEAD][RK];
    static_for<AHEAD>([&](auto a) {
      const int64_t at = (int64_t)(s + a) * 32 + fg * 8;
      const bool ok = s + a < s1 && at < p.k;
      static_for<RB>([&](auto i) { xv[a][i] = ok ? *reinterpret_cast<const v4i*>(xr[i] + at) : v4i{}; });
      static_for<RK>([&](auto j) { av[a][j] = ok && used[j] ? *reinterpret_cast<const v4i*>(ar[j] + at) : v4i{}; });
    });
    static_for<AHEAD>([&](auto a) {
      static_for<RB>([&](auto i) {
        static_for<RK>([&](auto j) { acc[i][j] = mfma16<F16>(av[a][j], xv[a][i], acc[i][j]); });
      });
    });
  }
  static_for<RB>([&](auto i) { static_for<RK>([&](auto j) { part[wave][i * RK + j][lane] = acc[i][j]; }); });
  __syncthreads();
  // Lane (fr, fg) of block (i, j): t of row i * 16 + fr, ranks r0 + j * 16 + 4 fg + 0 .. 3.
  for (int b = wave; b < RB * RK; b += RD_WAVES) {
    const int i = b / RK, j = b % RK, r = r0 + j * 16;
    if (r >= all || i * 16 + fr >= it.count) continue;
    v4f sum = part[0][b][lane];
    static_for<RD_WAVES - 1>([&](auto w) { sum += part[w + 1][b][lane]; });
    *reinterpret_cast<v4f*>(p.t + ((int64_t)blockIdx.y * p.rows + rows[i * 16 + fr]) * all + r + 4 * fg) = sum;
  }
}

// Tiles of 64 columns of one item.  MFMA block j of a tile holds the columns 16 g + 4 j + e in its rows 4 g + e, so that a
// lane ends with 16 columns of one row next to each other.
template <bool F16, int RB>
__global__ void __launch_bounds__(64 * RU_WAVES) request_up(const RequestAdapterParams p, int tiles_per_wave) {
  __shared__ int rows[RB * 16];
  const RequestItem it = request_item(p, (int)blockIdx.x, rows);
  if (it.count == 0) return;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int total = p.tiles[p.branches - 1], all = p.branches * p.width;
  const int rank = it.adapter < 0 ? 0 : p.ranks[it.adapter];
  const int begin = ((int)blockIdx.y * RU_WAVES + wave) * tiles_per_wave, end = min(begin + tiles_per_wave, total);
  for (int tile = begin; tile < end; ++tile) {
    int branch = 0;
    while (branch + 1 < p.branches && tile >= p.tiles[branch]) ++branch;
    const int n0 = (branch ? p.ends[branch - 1] : 0) + (tile - (branch ? p.tiles[branch - 1] : 0)) * 64;
    const int stop = p.ends[branch], n = n0 + 16 * fg;  // this lane's columns: n .. n + 15, up to stop
    v4f acc[RB][4];
    static_for<RB>([&](auto i) { static_for<4>([&](auto j) { acc[i][j] = v4f{}; }); });
    // Ranks r .. r + 7 of row block i, scaled; zeros past the rank.
    const float scaling = it.adapter < 0 ? 0.0f : p.scaling[it.adapter * p.branches + branch];
    auto low = [&](int i, int r, float (&v)[8]) {
      const float* src = p.t + (int64_t)rows[min(i * 16 + fr, it.count - 1)] * all + branch * p.width + min(r, p.width - 8);
      v4f x[2] = {v4f{}, v4f{}};
      for (int s = 0; s < p.splits; ++s) {
        x[0] += *reinterpret_cast<const v4f*>(src);
        x[1] += *reinterpret_cast<const v4f*>(src + 4);
        src += p.rows * all;
      }
      static_for<8>([&](auto e) { v[e] = r + e < rank ? x[e / 4][(int)(e % 4)] * scaling : 0.0f; });
    };
    // binary16 has not t's range: a row enters with its largest value in [1, 2).
    int shift[RB];
    static_for<RB>([&](auto i) {
      shift[i] = 0;
      if (!F16 || i * 16 >= it.count) return;
      float top = 0;
      for (int c0 = 0; c0 < rank; c0 += 32) {
        float v[8];
        low(i, c0 + 8 * fg, v);
        static_for<8>([&](auto e) { top = nan_max(top, fabsf(v[e])); });
      }
      top = nan_max(top, __shfl_xor(top, 16, 64));
      top = nan_max(top, __shfl_xor(top, 32, 64));
      const int exponent = (int)(__float_as_uint(top) >> 23);
      if (exponent < 255) shift[i] = exponent - 127;
    });
    for (int c0 = 0; c0 < rank; c0 += 32) {
      const int r = c0 + 8 * fg;
      v4i b[4];
      static_for<4>([&](auto j) {
        const int col = n0 + 16 * (fr >> 2) + 4 * j + (fr & 3);
        b[j] = r < p.width && col < stop
                   ? *reinterpret_cast<const v4i*>(p.up + ((int64_t)it.adapter * p.n + col) * p.width + r) : v4i{};
      });
      static_for<RB>([&](auto i) {
        if (i * 16 >= it.count) return;
        float v[8];
        low(i, r, v);
        v4i hi, lo;
        static_for<4>([&](auto e) {
          if constexpr (F16) static_for<2>([&](auto h) { v[2 * e + h] = __builtin_ldexpf(v[2 * e + h], -shift[i]); });
          hi[(int)e] = pack<F16>(v[2 * e], v[2 * e + 1]);
          float d[2];
          static_for<2>([&](auto h) {
            const float w = widen<F16>((uint32_t)hi[(int)e], h);
            d[h] = fabsf(w) < __builtin_inff() ? v[2 * e + h] - w : 0.0f;
          });
          lo[(int)e] = pack<F16>(d[0], d[1]);
        });
        static_for<4>([&](auto j) {
          acc[i][j] = mfma16<F16>(b[j], hi, acc[i][j]);
          acc[i][j] = mfma16<F16>(b[j], lo, acc[i][j]);
        });
      });
    }
    if constexpr (F16)
      static_for<RB>([&](auto i) {
        static_for<4>([&](auto j) { static_for<4>([&](auto e) { acc[i][j][(int)e] = __builtin_ldexpf(acc[i][j][(int)e], shift[i]); }); });
      });
    static_for<RB>([&](auto i) {
      if (i * 16 + fr >= it.count) return;
      const int64_t row = rows[i * 16 + fr];
      static_for<2>([&](auto h) {
        if (n + 8 * h >= stop) return;
        const v4i base = *reinterpret_cast<const v4i*>(p.base + row * p.ldb + n + 8 * h);
        v4i o;
        static_for<4>([&](auto e) {
          constexpr int at = 8 * h + 2 * e;
          const uint32_t w = (uint32_t)base[(int)e];
          o[(int)e] = pack<F16>(widen<F16>(w, 0) + acc[i][at / 4][at % 4], widen<F16>(w, 1) + acc[i][at / 4][at % 4 + 1]);
        });
        *reinterpret_cast<v4i*>(p.out + row * p.ldo + n + 8 * h) = rank > 0 ? o : base;
      });
    });
  }
}

// The launch of a call, from its sizes alone.
void request_plan(RequestAdapterParams& p) {
  const int64_t cus = compute_units();
  p.item_rows = p.rows > 512 ? 64 : 16;
  const int64_t groups = p.rows < p.adapters + 1 ? p.rows : p.adapters + 1;
  p.items = (int)(p.rows / p.item_rows + groups);
  if (p.items > p.rows) p.items = (int)p.rows;
  const int64_t steps = (p.k + 31) / 32, blocks = (p.branches * p.width + 63) / 64;
  // About one workgroup a CU, of at least two steps a wave.
  int64_t splits = cus / (p.items * blocks);
  if (splits > steps / (2 * RD_WAVES)) splits = steps / (2 * RD_WAVES);
  if (splits < 1) splits = 1;
  p.steps = (int)((steps + splits - 1) / splits);
  p.splits = (int)((steps + p.steps - 1) / p.steps);
}

int64_t request_workspace(const RequestAdapterParams& params) {
  RequestAdapterParams p = params;
  request_plan(p);
  const int64_t grouped = p.rows > RA_WAVE_ROWS ? 4 * (p.rows + 3 * (int64_t)p.items) : 0;
  return 4 * p.splits * p.rows * p.branches * p.width + grouped;
}

hipError_t launch_request_adapters(const RequestAdapterParams& params, bool f16, void* workspace, hipStream_t s) {
  RequestAdapterParams p = params;
  request_plan(p);
  p.t = static_cast<float*>(workspace);
  p.order = p.list = nullptr;
  if (p.rows > RA_WAVE_ROWS) {
    p.order = reinterpret_cast<int32_t*>(p.t + p.splits * p.rows * p.branches * p.width);
    p.list = p.order + p.rows;
    request_groups<<<1, 1024, 4 * (p.adapters + 1), s>>>(p);
  }
  int tiles = 0;
  for (int b = 0; b < p.branches; ++b) {
    tiles += (p.ends[b] - (b ? p.ends[b - 1] : 0) + 63) / 64;
    p.tiles[b] = tiles;
  }
  const int per = p.item_rows > 16 ? 4 : 1;
  const dim3 down((unsigned)p.items, (unsigned)p.splits, (unsigned)((p.branches * p.width + 63) / 64));
  const dim3 up((unsigned)p.items, (unsigned)((tiles + RU_WAVES * per - 1) / (RU_WAVES * per)));
  auto run = [&](auto type, auto blocks) {
    constexpr bool F16 = type;
    constexpr int RB = blocks;
    request_down<F16, RB, 4><<<down, 64 * RD_WAVES, 0, s>>>(p);
    request_up<F16, RB><<<up, 64 * RU_WAVES, 0, s>>>(p, per);
  };
  auto typed = [&](auto type) {
    if (p.item_rows > 16) run(type, std::integral_constant<int, 4>{});
    else run(type, std::integral_constant<int, 1>{});
  };
  if (f16) typed(std::true_type{});
  else typed(std::false_type{});
  return hipGetLastError();
}

}  // namespace vfa
