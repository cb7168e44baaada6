// The forms of the product with affine weights for few rows.
#pragma once

#include "few_core.h"

namespace mgq {

// X(number, NP, NQ, NE, waves, waves along the contraction, steps in flight + 1, us of a
// step for a wave alone on its SIMD, for waves that share it): 16 NQ entries (4 where NE
// = 1) by 16 NP rows for each of the waves that do not share them.
#define MGQ_AFFINE_SHAPES(X)             \
  X(1, 2, 1, 1, 4, 4, 3, 0.83, 0.55)     \
  X(2, 1, 1, 1, 8, 8, 3, 0.55, 0.38)     \
  X(3, 2, 1, 4, 4, 4, 2, 1.05, 0.79)     \
  X(4, 4, 1, 4, 4, 4, 2, 1.35, 1.27)     \
  X(5, 1, 1, 4, 8, 8, 3, 0.75, 0.58)     \
  X(6, 2, 1, 4, 4, 1, 2, 0.90, 0.45)     \
  X(7, 2, 1, 4, 4, 2, 2, 0.90, 0.45)     \
  X(8, 2, 2, 4, 4, 4, 2, 1.25, 1.31)     \
  X(9, 4, 2, 4, 4, 4, 2, 1.80, 2.00)     \
  X(10, 4, 4, 4, 4, 4, 2, 2.90, 3.00)    \
  X(11, 4, 2, 4, 4, 1, 2, 1.68, 1.68)

int affine_few_bits2(const LinArgs& a, const FewWeight& w, int choice, hipStream_t s, const char* what);
int affine_few_bits4(const LinArgs& a, const FewWeight& w, int choice, hipStream_t s, const char* what);
int affine_few_bits8(const LinArgs& a, const FewWeight& w, int choice, hipStream_t s, const char* what);

}  // namespace mgq
