// Few rows times affine weights of 2 bits.
#include "affine_few.h"

namespace mgq {

int affine_few_bits2(const LinArgs& a, const FewWeight& w, int choice, hipStream_t s, const char* what) {
  return run_types<kFewAf2>(a, w, choice, s, what);
}

}  // namespace mgq
