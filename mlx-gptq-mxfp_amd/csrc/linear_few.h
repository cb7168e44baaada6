// Products of few rows (linear_few.hip): forward only, any alignment.
#pragma once

#include "linear_tile.h"

namespace mgq {

// The low bits of where the operands' rows start and end (n bytes each).
inline uintptr_t lin_row_bounds(const LinArgs& a, int64_t n) {
  return reinterpret_cast<uintptr_t>(a.P) | reinterpret_cast<uintptr_t>(a.Q) |
         static_cast<uintptr_t>(a.ldp | a.ldq | a.p_group | n);
}
// A workgroup computes 16 nq entries (nq = 1, 2 or 4) by lin_few_cols(nq) weight rows.
inline int lin_few_cols(int nq) { return nq == 4 ? 32 : 16; }
inline int64_t lin_few_grid(const LinArgs& a, int nq) {
  return lin_row_tiles(a, 16 * nq) * ceil_div(a.np, lin_few_cols(nq));
}
constexpr int64_t kLinFewGrid = int64_t(1) << 24;  // 256 threads each, less than 2^32 in all
int lin_few_rows(const LinArgs& a, int op, int nq, hipStream_t s, const char* what);

}  // namespace mgq
