// Parameter block of the request adapters (not part of the C-ABI).
#pragma once
#include <stdint.h>

namespace vfa {

constexpr int RA_BRANCHES = 3, RA_ROWS = 16;
// Up to here every wave finds its rows itself; above, a launch of its own groups them.
constexpr int RA_WAVE_ROWS = 64;

struct RequestAdapterParams {
  const uint16_t *x, *base, *down, *up;
  uint16_t* out;
  int64_t ldx, ldb, ldo;
  const float* scaling;  // [adapters][branches]
  const int32_t* ranks;  // [adapters]
  const int64_t* index;  // [rows]
  int64_t rows, k, n;
  int adapters, branches, width;
  int ends[RA_BRANCHES];   // columns at which the branches end
  int groups[RA_BRANCHES];  // of columns, a workgroup's each, up to and with each branch
  int splits, steps;       // of K; 32-wide steps of a split
  int items, item_rows;    // at most; rows of one
  float* t;                // [splits][rows][branches * width]
  int32_t *order, *list;   // [items][item_rows] rows; [items][4]: adapter, count, rank
  int32_t* before;         // [rows] rows of the same adapter before
};

}  // namespace vfa
