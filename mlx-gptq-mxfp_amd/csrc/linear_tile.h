// The large-tile kernels' host side (linear_tile.hip) and wgrad's work list.
#pragma once

#include "linear_common.h"

namespace mgq {

enum LinKind : int { kLinForward = 0, kLinDgrad = 1, kLinWgrad = 2, kLinWgradGather = 3 };

// wgrad: group g's entries [t0, t1). slot >= 0: the group is cut and the unit's
// tile `i` goes to partial tile slot * tiles + i.
struct LinUnit {
  int32_t g, t0, t1, slot;
};
// A cut group: its units' slots are slot0 .. slot0 + n - 1.
struct LinSplit {
  int32_t g, slot0, n;
};
struct LinPlanArgs {
  int32_t* counts;  // units, cut groups
  LinUnit* units;
  LinSplit* splits;
  float* partials;
  int npt, nqt, bq;
  int cap;
  int max_units, max_splits, max_slots;
  int deal;  // whole units per XCD
};
struct LinPlanSizes {
  int64_t tiles, cap, max_units, max_splits, max_slots;
  int64_t units_off, splits_off, partials_off, bytes;
};
constexpr int kLinPlanGroups = 4096;

// wgrad: which unit and tile an item is: 1 if there is one, 0 past the last, -1 for a
// hole in the order. With many units an XCD takes every eighth of them whole (in
// snake order: they are sorted by length), so that its L2 holds the unit's rows;
// with few, a unit's tiles go round the XCDs.
__device__ __forceinline__ int lin_find_unit(const LinArgs& a, const LinPlanArgs& pl, uint32_t item,
                                             LinUnit* u, int* tile) {
  const uint32_t tiles = static_cast<uint32_t>(pl.npt) * pl.nqt;
  const int n = pl.counts[0];
  int i;
  if (pl.deal) {
    const uint32_t x = item & 7, j = item >> 3;
    const uint32_t round = j / tiles;
    *tile = static_cast<int>(j % tiles);
    i = static_cast<int>(round * 8 + (round & 1 ? 7 - x : x));
    if (i >= n) return static_cast<int>(round * 8) >= n ? 0 : -1;
  } else {
    i = static_cast<int>(item / tiles);
    *tile = static_cast<int>(item % tiles);
    if (i >= n) return 0;
  }
  const LinUnit v = pl.units[i];
  u->g = __builtin_amdgcn_readfirstlane(v.g);
  u->t0 = __builtin_amdgcn_readfirstlane(v.t0);
  u->t1 = __builtin_amdgcn_readfirstlane(v.t1);
  u->slot = __builtin_amdgcn_readfirstlane(v.slot);
  if (u->slot >= 0) u->slot = u->slot * static_cast<int>(tiles) + *tile;
  return 1;
}

// The host's bound on the row tiles of a launch.
inline int64_t lin_row_tiles(const LinArgs& a, int bm) {
  const int64_t segs = a.G + 2;
  return a.offsets ? a.M / bm + (segs < a.M ? segs : a.M) : ceil_div(a.M, bm);
}

inline int64_t lin_tile_grid(const LinArgs& a, int rows, int cols) {
  return lin_row_tiles(a, rows) * ceil_div(a.np, cols);
}
constexpr int64_t kLinTileGrid = int64_t(1) << 23;  // 512 threads each, less than 2^32 in all

// Output tile of a product over rows: 64, 128 or 256 entries by 256 columns, or
// 64 by 128. staged: through registers (up to 128 entries).
struct LinTileShape {
  int rows, cols;
  bool staged;
};

// Whether the operands' rows start and end on 16-byte boundaries.
bool lin_tile_direct(const LinArgs& a, int op, int kind);
int lin_tile_rows(const LinArgs& a, int op, int kind, LinTileShape t, hipStream_t s,
                  const char* what);
int64_t lin_tile_wgrad_bytes(int64_t M, int64_t G, int64_t N, int64_t K);
int lin_tile_wgrad(const LinArgs& a, int op, void* workspace, hipStream_t s, const char* what);

}  // namespace mgq
