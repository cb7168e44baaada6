// Products of few rows (linear_few.hip): forward only, any alignment.
#pragma once

#include "linear_tile.h"

namespace mgq {

// The low bits of where the operands' rows start and end (n bytes each).
inline uintptr_t lin_row_bounds(const LinArgs& a, int64_t n) {
  return reinterpret_cast<uintptr_t>(a.P) | reinterpret_cast<uintptr_t>(a.Q) |
         static_cast<uintptr_t>(a.ldp | a.ldq | a.p_group | n);
}
int lin_few_rows(const LinArgs& a, int op, int nq, hipStream_t s, const char* what);

}  // namespace mgq
