// The low-rank adapters of many requests beside a shared projection, for gfx950:
//   out[m] = base[m] + scaling[i][b] (x[m] A_i^T) B_i^T,  i = index[m] (none outside [0, adapters): out[m] = base[m]),
// column n taking branch b's part of A_i (the branches of a merged projection).
//
// Rows are taken by adapter, whatever their order: an item is up to 16 (or 64) rows of one adapter, so each
// adapter in use is read about once.  Two products on the matrix cores, v_mfma_f32_16x16x32 with the
// adapter's rows as operand A and the items' rows as operand B:
//   request_down  t = x A^T, binary32.  K is split over the waves of a workgroup and, where there are few items, over
//                 workgroups.
//   request_up    adds the splits up in their order, keeps t of its item in LDS as two bf16, a high and a low part (16
//                 bits of it or more, in binary32's range), and multiplies by B.  Binary16 factors of B are two bf16
//                 as well, exactly.  scaling, base and one rounding follow.
// Few rows of short inputs take both in one launch, request_few.
// Nothing is added by atomics: a row's result does not depend on its company.
// Bound by launches for a few rows, by the adapters' bytes for a decoding batch, and by base and out for prompts.
#include "request_adapters.h"

#include <type_traits>

#include "common.h"

namespace vfa {

int compute_units();

namespace {

typedef int v2i __attribute__((ext_vector_type(2)));
constexpr int RD_WAVES = 8;  // of request_down: parts of K
constexpr int RU_WAVES = 4;  // of request_up: column tiles

struct RequestItem {
  int adapter, count, rank;  // adapter -1: none; count 0: no such item
};

__device__ __forceinline__ int rank_of(const RequestAdapterParams& p, int adapter) {
  return max(0, min(p.ranks[adapter], p.width));
}

// Item `index` of at most 64 rows, found by the wave: the adapters by their first row, their rows in order.
__device__ __forceinline__ RequestItem request_find(const RequestAdapterParams& p, int index, int* rows) {
  const int lane = (int)threadIdx.x & 63;
  int mine = -2, rank = 0;  // no row
  // The ranks of up to 64 adapters come with the indices instead of after them.
  const bool few = p.adapters <= 64;
  const int ranks = few && lane < p.adapters ? rank_of(p, lane) : 0;
  if (lane < p.rows) {
    const int64_t i = p.index[lane];
    mine = (uint64_t)i < (uint64_t)p.adapters ? (int)i : -1;
    if (mine >= 0 && !few) rank = rank_of(p, mine);
  }
  if (few) rank = __shfl(ranks, max(mine, 0), 64);
  uint64_t left = __builtin_amdgcn_ballot_w64(mine != -2);
  while (left) {
    const int first = __builtin_ctzll(left), a = __builtin_amdgcn_readlane(mine, first);
    const uint64_t same = __builtin_amdgcn_ballot_w64(mine == a);
    const int count = __popcll(same), items = (count + p.item_rows - 1) / p.item_rows;
    if (index < items) {
      // Lane l of the adapter's rows goes to its place among them.
      const int place = __popcll(same & ((uint64_t(1) << lane) - 1)) - index * p.item_rows;
      if (mine == a && place >= 0 && place < p.item_rows) rows[place] = lane;
      return RequestItem{a, min(p.item_rows, count - index * p.item_rows), a < 0 ? 0 : __builtin_amdgcn_readlane(rank, first)};
    }
    index -= items;
    left &= ~same;
  }
  return RequestItem{-1, 0, 0};
}

// Item `index` as request_groups or request_down left it, its rows in `rows` (LDS of this workgroup).
__device__ __forceinline__ RequestItem request_listed(const RequestAdapterParams& p, int index, int* rows) {
  const v4i item = *reinterpret_cast<const v4i*>(p.list + 4 * index);
  if ((int)threadIdx.x < p.item_rows) rows[threadIdx.x] = p.order[(int64_t)index * p.item_rows + threadIdx.x];
  return RequestItem{item[0], item[1], item[2]};
}

__device__ __forceinline__ RequestItem uniform(const RequestItem& it) {
  return RequestItem{__builtin_amdgcn_readfirstlane(it.adapter), __builtin_amdgcn_readfirstlane(it.count),
                     __builtin_amdgcn_readfirstlane(it.rank)};
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
// Two values as bf16 and what that leaves of them, as bf16.  An infinity leaves nothing.
__device__ __forceinline__ void parts(float a, float b, int& high, int& low) {
  high = pack<false>(a, b);
  const float x = bf16_lo((uint32_t)high), y = bf16_hi((uint32_t)high);
  low = pack<false>(fabsf(x) < __builtin_inff() ? a - x : 0.0f, fabsf(y) < __builtin_inff() ? b - y : 0.0f);
}

// Eight bf16, zeros in the place of those that are not finite.
__device__ __forceinline__ v4i finite(v4i w) {
  static_for<4>([&](auto i) {
    const uint32_t u = (uint32_t)w[(int)i];
    w[(int)i] = (int)(((u & 0x7f80u) == 0x7f80u ? 0 : u & 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0 : u & 0xffff0000u));
  });
  return w;
}

__device__ __forceinline__ int wave_sum_before(int v, int lane) {  // inclusive
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

}  // namespace

// The items of more than 64 rows, by adapter, those without one last.  One workgroup: a histogram, its prefix sums,
// and the rows to their places (within an adapter in any order: no row's result depends on it).
__global__ void __launch_bounds__(1024) request_groups(const RequestAdapterParams p) {
  extern __shared__ int counts[];  // [adapters + 1]: rows, then the first place in p.order
  __shared__ int sums[17];
  const int bins = p.adapters + 1, t = (int)threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int b = t; b < bins; b += 1024) counts[b] = 0;
  // Thread t's bins are next to each other; their ranks are on the way meanwhile.
  const int per = (bins + 1023) / 1024, b0 = min(t * per, bins), b1 = min(b0 + per, bins);
  const int rank0 = b0 < p.adapters ? rank_of(p, b0) : 0;
  __syncthreads();
  auto bin_of = [&](int64_t m) {
    if (m >= p.rows) return -1;
    const int64_t i = p.index[m];
    return (uint64_t)i < (uint64_t)p.adapters ? (int)i : p.adapters;
  };
  // Adds one to a bin for each lane, and gives each the count before it.  Lanes of one bin (runs) go together, for the first
  // two bins of a wave: the same word is added to once at a time.
  auto add = [&](int bin) {
    int before = 0;
    uint64_t left = __builtin_amdgcn_ballot_w64(bin >= 0);
    for (int i = 0; i < 2 && left; ++i) {
      const int first = __builtin_ctzll(left), b = __builtin_amdgcn_readlane(bin, first);
      const uint64_t same = __builtin_amdgcn_ballot_w64(bin == b);
      int old = 0;
      if (lane == first) old = atomicAdd(&counts[b], __popcll(same));
      old = __builtin_amdgcn_readlane(old, first);
      if (bin == b) before = old + __popcll(same & ((uint64_t(1) << lane) - 1));
      left &= ~same;
    }
    if (left >> lane & 1) before = atomicAdd(&counts[bin], 1);
    return before;
  };
  // The first rows of each thread stay in registers.
  constexpr int KEPT = 8;
  int bins_of[KEPT], before_of[KEPT];
  static_for<KEPT>([&](auto i) { bins_of[i] = bin_of(t + 1024 * i); });
  static_for<KEPT>([&](auto i) {
    if (1024 * i < p.rows) before_of[i] = add(bins_of[i]);
  });
  const int64_t end = (p.rows + 1023) / 1024 * 1024;
  for (int64_t m = t + 1024 * KEPT; m < end; m += 1024) {
    const int before = add(bin_of(m));
    if (m < p.rows) p.before[m] = before;
  }
  __syncthreads();
  auto items_of = [&](int c) { return (c + p.item_rows - 1) / p.item_rows; };
  int items = 0;
  for (int b = b0; b < b1; ++b) items += items_of(counts[b]);
  int item = wave_sum_before(items, lane);
  if (lane == 63) sums[wave] = item;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) item += sums[w];
    all += sums[w];
  }
  item -= items;
  for (int b = b0; b < b1; ++b) {
    const int c = counts[b], rank = b == b0 ? rank0 : b < p.adapters && c ? rank_of(p, b) : 0;
    counts[b] = item * p.item_rows;
    for (int first = 0; first < c; first += p.item_rows, ++item)
      *reinterpret_cast<v4i*>(p.list + 4 * item) = v4i{b < p.adapters ? b : -1, min(p.item_rows, c - first), rank, 0};
  }
  for (int i = all + t; i < p.items; i += 1024) *reinterpret_cast<v4i*>(p.list + 4 * i) = v4i{};
  __syncthreads();
  static_for<KEPT>([&](auto i) {
    if (bins_of[i] >= 0) p.order[counts[bins_of[i]] + before_of[i]] = t + 1024 * i;
  });
  for (int64_t m = t + 1024 * KEPT; m < p.rows; m += 1024) p.order[counts[bin_of(m)] + p.before[m]] = (int)m;
}

// t of an item's RB blocks of 16 rows for RK blocks of 16 adapter rows and one split of K.  Items of 64 rows read A
// once for all four blocks: a workgroup for each 16 took 51 us for 1000 rows of 24 adapters (rank 64, K 5120, three
// branches), bound by what L2 delivers.
template <bool F16, int RB, int RK>
__global__ void __launch_bounds__(64 * RD_WAVES) request_down(const RequestAdapterParams p) {
  constexpr int PASS = RB > 2 ? 2 : RB;  // row blocks whose sums are in LDS together
  __shared__ int rows[RB * 16];
  __shared__ v4f part[RD_WAVES][PASS * RK][64];
  const int item = (int)blockIdx.x;
  const bool grouped = p.rows > RA_WAVE_ROWS;
  // Ungrouped, every wave finds the same and writes the same.
  const RequestItem it = uniform(grouped ? request_listed(p, item, rows) : request_find(p, item, rows));
  __syncthreads();
  if (!grouped && blockIdx.y == 0 && blockIdx.z == 0) {  // for request_up
    if (threadIdx.x == 0) *reinterpret_cast<v4i*>(p.list + 4 * item) = v4i{it.adapter, it.count, it.rank, 0};
    if ((int)threadIdx.x < it.count) p.order[item * p.item_rows + threadIdx.x] = rows[threadIdx.x];
  }
  if (it.count == 0 || it.adapter < 0) return;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int all = p.branches * p.width, r0 = (int)blockIdx.z * RK * 16;

  // Blocks of adapter rows that hold some of the rank.
  bool used[RK], any = false;
  const uint16_t *xr[RB], *ar[RK];
  static_for<RK>([&](auto j) {
    const int r = r0 + j * 16;
    used[j] = r < all && r % p.width < it.rank;
    any = any || used[j];
    ar[j] = p.down + ((int64_t)it.adapter * all + min(r + fr, all - 1)) * p.k;
  });
  if (!any) return;
  static_for<RB>([&](auto i) { xr[i] = p.x + (int64_t)rows[min((int)i * 16 + fr, it.count - 1)] * p.ldx; });
  const int steps = (int)((p.k + 31) / 32);
  const int from = (int)blockIdx.y * p.steps, to = min(from + p.steps, steps);
  const int s0 = from + max(0, to - from) * wave / RD_WAVES, s1 = from + max(0, to - from) * (wave + 1) / RD_WAVES;

  constexpr int AHEAD = RB == 1 || RK <= 2 ? 8 : 4;  // steps whose loads are in flight together
  v4f acc[RB][RK];
  static_for<RB>([&](auto i) { static_for<RK>([&](auto j) { acc[i][j] = v4f{}; }); });
  for (int s = s0; s < s1; s += AHEAD) {
    v4i xv[AHEAD][RB], av[AHEAD][RK];
    static_for<AHEAD>([&](auto a) {
      const int64_t at = (int64_t)(s + a) * 32 + fg * 8;
      const bool ok = s + a < s1 && at < p.k;
      static_for<RB>([&](auto i) { xv[a][i] = ok && i * 16 < it.count ? *reinterpret_cast<const v4i*>(xr[i] + at) : v4i{}; });
      static_for<RK>([&](auto j) { av[a][j] = ok && used[j] ? *reinterpret_cast<const v4i*>(ar[j] + at) : v4i{}; });
    });
    static_for<AHEAD>([&](auto a) {
      static_for<RB>([&](auto i) {
        static_for<RK>([&](auto j) { acc[i][j] = mfma16<F16>(av[a][j], xv[a][i], acc[i][j]); });
      });
    });
  }
  static_for<RB / PASS>([&](auto pass) {
    if (pass) __syncthreads();
    static_for<PASS>([&](auto i) { static_for<RK>([&](auto j) { part[wave][i * RK + j][lane] = acc[pass * PASS + i][j]; }); });
    __syncthreads();
    // Lane (fr, fg) of block (i, j): t of row i * 16 + fr, ranks r0 + j * 16 + 4 fg + 0 .. 3.
    for (int b = wave; b < PASS * RK; b += RD_WAVES) {
      const int i = pass * PASS + b / RK, r = r0 + b % RK * 16;
      if (r >= all || i * 16 + fr >= it.count) continue;
      v4f sum = part[0][b][lane];
      static_for<RD_WAVES - 1>([&](auto w) { sum += part[w + 1][b][lane]; });
      *reinterpret_cast<v4f*>(p.t + ((int64_t)blockIdx.y * p.rows + rows[i * 16 + fr]) * all + r + 4 * fg) = sum;
    }
  });
}

namespace {

// A branch's columns: those of workgroup `group` of the call's groups.
struct RequestColumns {
  int branch, group, first, stop;
};
__device__ __forceinline__ RequestColumns request_columns(const RequestAdapterParams& p, int group) {
  int branch = 0;
  while (branch + 1 < p.branches && group >= p.groups[branch]) ++branch;
  if (branch) group -= p.groups[branch - 1];
  return RequestColumns{branch, group, branch ? p.ends[branch - 1] : 0, p.ends[branch]};
}

// A wave's tile of 64 columns of one branch and item (RB blocks of 16 rows), ranks in NC runs of 32.  MFMA block j
// holds the columns 32 (j / 2) + 8 g + 4 (j % 2) + e in its rows 4 g + e, so that a lane ends with two runs of eight columns
// of one row, and the four lanes of a row store 64 bytes at once.
template <bool F16, int RB, int NC>
struct RequestTile {
  static constexpr int PITCH = 64 * NC + 8;  // of a row in LDS: high parts, low parts, and eight against bank conflicts
  v4i b[NC][4], base[RB][2];
  int64_t row[RB];

  __device__ __forceinline__ void load(const RequestAdapterParams& p, const RequestItem& it, const int* rows, int n0, int stop) {
    const int lane = (int)threadIdx.x & 63, fr = lane & 15, fg = lane >> 4;
    const int n = n0 + 8 * fg;  // this lane's columns: n .. n + 7 and 32 further, up to stop
    static_for<NC>([&](auto c) {
      const int r = c * 32 + 8 * fg;
      static_for<4>([&](auto j) {
        const int col = n0 + 32 * (j / 2) + 8 * (fr >> 2) + 4 * (j % 2) + (fr & 3);
        b[c][j] = r < it.rank && col < stop
                      ? *reinterpret_cast<const v4i*>(p.up + ((int64_t)it.adapter * p.n + col) * p.width + r) : v4i{};
      });
    });
    static_for<RB>([&](auto i) {
      if (16 * i >= it.count) return;
      row[i] = rows[min(16 * (int)i + fr, it.count - 1)];
      static_for<2>([&](auto h) {
        base[i][h] = n + 32 * h < stop ? *reinterpret_cast<const v4i*>(p.base + row[i] * p.ldb + n + 32 * h) : v4i{};
      });
    });
  }

  __device__ __forceinline__ void store(const RequestAdapterParams& p, const RequestItem& it, const uint16_t* low_rank,
                                        float scaling, int n0, int stop) {
    const int lane = (int)threadIdx.x & 63, fr = lane & 15, fg = lane >> 4;
    const int n = n0 + 8 * fg;
    v4i rest[NC][4];
    if constexpr (F16)
      static_for<NC>([&](auto c) {
        static_for<4>([&](auto j) {
          static_for<4>([&](auto e) {
            const uint32_t w = (uint32_t)b[c][j][(int)e];
            int high, low;
            parts(widen<true>(w, 0), widen<true>(w, 1), high, low);
            b[c][j][(int)e] = high;
            rest[c][j][(int)e] = low;
          });
        });
      });
    static_for<RB>([&](auto i) {
      if (16 * i >= it.count) return;
      v4f acc[4];
      static_for<4>([&](auto j) { acc[j] = v4f{}; });
      const uint16_t* src = low_rank + min(16 * (int)i + fr, it.count - 1) * PITCH + 8 * fg;
      static_for<NC>([&](auto c) {
        if (c * 32 >= it.rank) return;
        const v4i high = *reinterpret_cast<const v4i*>(src + c * 32), low = *reinterpret_cast<const v4i*>(src + 32 * NC + c * 32);
        static_for<4>([&](auto j) {
          acc[j] = mfma16<false>(b[c][j], high, acc[j]);
          acc[j] = mfma16<false>(b[c][j], low, acc[j]);
        });
        if constexpr (F16) {
          const v4i near = finite(high);  // an infinity is in the first product
          static_for<4>([&](auto j) { acc[j] = mfma16<false>(rest[c][j], near, acc[j]); });
        }
      });
      if (16 * i + fr >= it.count) return;
      static_for<2>([&](auto h) {
        if (n + 32 * h >= stop) return;
        v4i o;
        static_for<4>([&](auto e) {
          constexpr int at = 8 * h + 2 * e;
          const uint32_t w = (uint32_t)base[i][h][(int)e];
          o[(int)e] = pack<F16>(__builtin_fmaf(acc[at / 4][at % 4], scaling, widen<F16>(w, 0)),
                                __builtin_fmaf(acc[at / 4][at % 4 + 1], scaling, widen<F16>(w, 1)));
        });
        *reinterpret_cast<v4i*>(p.out + row[i] * p.ldo + n + 32 * h) = it.rank > 0 ? o : base[i][h];
      });
    });
  }
};

}  // namespace

// out from t, four tiles of columns and an item a workgroup.
template <bool F16, int NC>
__global__ void __launch_bounds__(64 * RU_WAVES) request_up(const RequestAdapterParams p) {
  using Tile = RequestTile<F16, 4, NC>;
  __shared__ int rows[64];
  __shared__ __attribute__((aligned(16))) uint16_t low_rank[64 * Tile::PITCH];
  const RequestItem it = uniform(request_listed(p, (int)blockIdx.y, rows));
  __syncthreads();
  if (it.count == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const RequestColumns columns = request_columns(p, (int)blockIdx.x);
  const float scaling = it.adapter < 0 ? 0.0f : p.scaling[it.adapter * p.branches + columns.branch];

  // t, eight ranks a thread; zeros past the rank.
  if (it.rank > 0) {
    const int all = p.branches * p.width;
    for (int e = (int)threadIdx.x; e < it.count * 4 * NC; e += 64 * RU_WAVES) {
      const int row = e / (4 * NC), r = e % (4 * NC) * 8;
      v4f x[2] = {v4f{}, v4f{}};
      if (r < it.rank) {
        const float* src = p.t + (int64_t)rows[row] * all + columns.branch * p.width + r;
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s, src += p.rows * all) {
          x[0] += *reinterpret_cast<const v4f*>(src);
          x[1] += *reinterpret_cast<const v4f*>(src + 4);
        }
      }
      v4i high, low;
      static_for<4>([&](auto i) {
        int h, l;
        parts(r + 2 * i < it.rank ? x[i / 2][2 * (i % 2)] : 0.0f, r + 2 * i + 1 < it.rank ? x[i / 2][2 * (i % 2) + 1] : 0.0f, h, l);
        high[(int)i] = h;
        low[(int)i] = l;
      });
      *reinterpret_cast<v4i*>(low_rank + row * Tile::PITCH + r) = high;
      *reinterpret_cast<v4i*>(low_rank + row * Tile::PITCH + 32 * NC + r) = low;
    }
  }
  __syncthreads();

  const int n0 = columns.first + (columns.group * RU_WAVES + wave) * 64;
  if (n0 >= columns.stop) return;
  Tile tile;
  tile.load(p, it, rows, n0, columns.stop);
  tile.store(p, it, low_rank, scaling, n0, columns.stop);
}

// Both products in one launch, for up to 64 rows and small A: eight tiles of columns and an item of 16 rows a workgroup, each
// of which forms t of its branch for itself, RK blocks of 16 ranks.  x must not overlap out.
template <bool F16, int RK>
__global__ void __launch_bounds__(64 * RD_WAVES) request_few(const RequestAdapterParams p) {
  constexpr int NC = (RK + 1) / 2;
  using Tile = RequestTile<F16, 1, NC>;
  __shared__ int rows[16];
  __shared__ v4f part[RD_WAVES][RK][64];
  __shared__ __attribute__((aligned(16))) uint16_t low_rank[16 * Tile::PITCH];
  const RequestItem it = uniform(p.rows > RA_WAVE_ROWS ? request_listed(p, (int)blockIdx.y, rows) : request_find(p, (int)blockIdx.y, rows));
  __syncthreads();
  if (it.count == 0) return;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const RequestColumns columns = request_columns(p, (int)blockIdx.x);
  const int n0 = columns.first + (columns.group * RD_WAVES + wave) * 64;
  const float scaling = it.adapter < 0 ? 0.0f : p.scaling[it.adapter * p.branches + columns.branch];
  Tile tile;
  tile.load(p, it, rows, n0, columns.stop);  // on its way beside A and x
  if (it.rank > 0) {
    const uint16_t* xr = p.x + (int64_t)rows[min(fr, it.count - 1)] * p.ldx;
    const uint16_t* ar[RK];
    static_for<RK>([&](auto j) {
      ar[j] = p.down + (((int64_t)it.adapter * p.branches + columns.branch) * p.width + min(j * 16 + fr, p.width - 1)) * p.k;
    });
    const int steps = (int)((p.k + 31) / 32), s0 = steps * wave / RD_WAVES, s1 = steps * (wave + 1) / RD_WAVES;
    constexpr int AHEAD = RK == 1 ? 16 : 8;
    v4f acc[RK];
    static_for<RK>([&](auto j) { acc[j] = v4f{}; });
    for (int s = s0; s < s1; s += AHEAD) {
      v4i xv[AHEAD], av[AHEAD][RK];
      static_for<AHEAD>([&](auto a) {
        const int64_t at = (int64_t)(s + a) * 32 + fg * 8;
        const bool ok = s + a < s1 && at < p.k;
        xv[a] = ok ? *reinterpret_cast<const v4i*>(xr + at) : v4i{};
        static_for<RK>([&](auto j) { av[a][j] = ok && j * 16 < it.rank ? *reinterpret_cast<const v4i*>(ar[j] + at) : v4i{}; });
      });
      static_for<AHEAD>([&](auto a) { static_for<RK>([&](auto j) { acc[j] = mfma16<F16>(av[a][j], xv[a], acc[j]); }); });
    }
    static_for<RK>([&](auto j) { part[wave][j][lane] = acc[j]; });
    __syncthreads();
    // Wave j: t of row fr, ranks 16 j + 4 fg + 0 .. 3, zeros past the rank.
    if (wave < 2 * NC) {
      const int r = 16 * wave + 4 * fg;
      v4f sum = v4f{};
      if (wave < RK) static_for<RD_WAVES>([&](auto w) { sum += part[w][wave][lane]; });
      v2i high, low;
      static_for<2>([&](auto i) {
        int h, l;
        parts(r + 2 * i < it.rank ? sum[2 * i] : 0.0f, r + 2 * i + 1 < it.rank ? sum[2 * i + 1] : 0.0f, h, l);
        high[(int)i] = h;
        low[(int)i] = l;
      });
      *reinterpret_cast<v2i*>(low_rank + fr * Tile::PITCH + r) = high;
      *reinterpret_cast<v2i*>(low_rank + fr * Tile::PITCH + 32 * NC + r) = low;
    }
  }
  __syncthreads();
  if (n0 < columns.stop) tile.store(p, it, low_rank, scaling, n0, columns.stop);
}

namespace {

// Adapter rows that a workgroup of request_down takes.
int request_ranks(const RequestAdapterParams& p) {
  const int all = p.branches * p.width;
  return all >= 64 ? 64 : all >= 32 ? 32 : 16;
}

// The launch of a call, from its sizes alone.
void request_plan(RequestAdapterParams& p) {
  const int64_t cus = compute_units();
  // Items of 64 rows read A and B less often, those of 16 are more: us with 64 and with 16, K 5120: 256 rows of 24 adapters of
  // rank 64 beside three branches 28.8, 27.9, 400 rows 32.7, 40.7; of rank 32 beside one, 600 rows 20.5, 19.8, 1000 rows
  // 23.6, 26.1; 1000 rows of 4 adapters of rank 16 21.5, 19.1.
  p.item_rows = p.rows > 300 && p.rows * p.branches * p.width >= 24576 ? 64 : 16;
  const int64_t groups = p.rows < p.adapters + 1 ? p.rows : p.adapters + 1;
  p.items = (int)(p.rows / p.item_rows + groups);
  if (p.items > p.rows) p.items = (int)p.rows;
  const int64_t steps = (p.k + 31) / 32, blocks = (p.branches * p.width + request_ranks(p) - 1) / request_ranks(p);
  // About one workgroup a CU, of at least two steps a wave.
  int64_t splits = cus / (p.items * blocks);
  if (splits > steps / (2 * RD_WAVES)) splits = steps / (2 * RD_WAVES);
  if (splits < 1) splits = 1;
  p.steps = (int)((steps + splits - 1) / splits);
  p.splits = (int)((steps + p.steps - 1) / p.steps);
}

// Groups of `columns` columns of one branch.
int request_grouped(RequestAdapterParams& p, int columns) {
  int groups = 0;
  for (int b = 0; b < p.branches; ++b) {
    groups += (p.ends[b] - (b ? p.ends[b - 1] : 0) + columns - 1) / columns;
    p.groups[b] = groups;
  }
  return groups;
}

// Whether request_few takes the call: a launch less, but every workgroup reads A of its item and branch, of which a CU gets
// 33 bytes a ns.  us with and without, one projection: 1 row, K 1536, rank 16 6.6, 9.3, rank 32 8.6, 10.0, rank 64 11.7,
// 11.1; K 1024, rank 64 10.1, 10.9; K 5120, rank 16 10.7, 9.6.  40 rows of 20 adapters, K 1536, rank 32 12.0, 13.5.  100 rows of
// 4, K 1536, rank 16 11.1, 12.9, rank 32 13.4, 13.4; K 2048, rank 16 12.3, 11.4.  600 rows, 440 workgroups 17.3, 14.1.
bool request_alone(RequestAdapterParams& p) {
  const int64_t most = p.rows > RA_WAVE_ROWS ? 32768 : 65536;
  if (p.item_rows > 16 || p.width > 64 || p.k > 1536 || p.k * p.width > most) return false;
  if (4 * (int64_t)p.items * request_grouped(p, 64 * RD_WAVES) > 5 * compute_units()) return false;
  // Its workgroups read x while others write.
  const uint16_t *x = p.x, *x_end = x + (p.rows - 1) * p.ldx + p.k, *out = p.out, *out_end = out + (p.rows - 1) * p.ldo + p.n;
  return x_end <= out || out_end <= x;
}

// Values of t.
int64_t request_low_ranks(const RequestAdapterParams& p) { return (int64_t)p.splits * p.rows * p.branches * p.width; }

}  // namespace

int64_t request_workspace(const RequestAdapterParams& params) {
  RequestAdapterParams p = params;
  request_plan(p);
  return 4 * (request_low_ranks(p) + (int64_t)p.items * (4 + p.item_rows) + (p.rows > RA_WAVE_ROWS ? p.rows : 0));
}

hipError_t launch_request_adapters(const RequestAdapterParams& params, bool f16, void* workspace, hipStream_t s) {
  RequestAdapterParams p = params;
  request_plan(p);
  p.t = static_cast<float*>(workspace);
  p.list = reinterpret_cast<int32_t*>(p.t + request_low_ranks(p));
  p.order = p.list + 4 * (int64_t)p.items;
  p.before = p.order + (int64_t)p.items * p.item_rows;
  if (p.rows > RA_WAVE_ROWS) request_groups<<<1, 1024, 4 * (p.adapters + 1), s>>>(p);
  if (request_alone(p)) {
    const dim3 grid((unsigned)request_grouped(p, 64 * RD_WAVES), (unsigned)p.items);
    auto few = [&](auto type) {
      constexpr bool F16 = type;
      if (p.width <= 16) request_few<F16, 1><<<grid, 64 * RD_WAVES, 0, s>>>(p);
      else if (p.width <= 32) request_few<F16, 2><<<grid, 64 * RD_WAVES, 0, s>>>(p);
      else request_few<F16, 4><<<grid, 64 * RD_WAVES, 0, s>>>(p);
    };
    if (f16) few(std::true_type{});
    else few(std::false_type{});
    return hipGetLastError();
  }
  const int ranks = request_ranks(p), groups = request_grouped(p, 64 * RU_WAVES);
  const dim3 down((unsigned)p.items, (unsigned)p.splits, (unsigned)((p.branches * p.width + ranks - 1) / ranks));
  // An item's columns next to each other: 4093 rows 83.4 us, with the items next to each other 85.5.
  const dim3 up((unsigned)groups, (unsigned)p.items);
  auto run_down = [&](auto type, auto blocks) {
    constexpr bool F16 = type;
    constexpr int RB = blocks;
    if (ranks == 64) request_down<F16, RB, 4><<<down, 64 * RD_WAVES, 0, s>>>(p);
    else if (ranks == 32) request_down<F16, RB, 2><<<down, 64 * RD_WAVES, 0, s>>>(p);
    else request_down<F16, RB, 1><<<down, 64 * RD_WAVES, 0, s>>>(p);
  };
  auto typed = [&](auto type) {
    constexpr bool F16 = type;
    if (p.item_rows > 16) run_down(type, std::integral_constant<int, 4>{});
    else run_down(type, std::integral_constant<int, 1>{});
    if (p.width <= 32) request_up<F16, 1><<<up, 64 * RU_WAVES, 0, s>>>(p);
    else if (p.width <= 64) request_up<F16, 2><<<up, 64 * RU_WAVES, 0, s>>>(p);
    else request_up<F16, 4><<<up, 64 * RU_WAVES, 0, s>>>(p);
  };
  if (f16) typed(std::true_type{});
  else typed(std::false_type{});
  return hipGetLastError();
}

}  // namespace vfa
