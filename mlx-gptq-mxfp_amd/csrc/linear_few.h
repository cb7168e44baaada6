// Products of few rows (linear_few.hip): forward only, any alignment.
#pragma once

#include "linear_tile.h"

namespace mgq {

int lin_few_rows(const LinArgs& a, int op, int nq, hipStream_t s, const char* what);

}  // namespace mgq
