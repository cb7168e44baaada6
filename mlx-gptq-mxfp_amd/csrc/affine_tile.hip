// The tile kernel (linear_tile_kernel.h) with affine weights: codes stay codes in LDS, with
// the scale and the bias of each row and half stage, and become q s + b, rounded to the
// rows' type, in registers.
#include "linear_tile_kernel.h"

namespace mgq {

int lin_tile_affine(const LinArgs& a, int op, LinTileShape t, hipStream_t s, const char* what) {
  switch (op) {
    case kOpAf2: return pick_rows<kOpAf2, kLinForward>(a, t, s, what);
    case kOpAf4: return pick_rows<kOpAf4, kLinForward>(a, t, s, what);
    case kOpAf8: return pick_rows<kOpAf8, kLinForward>(a, t, s, what);
    case kOpAf2H: return pick_rows<kOpAf2H, kLinForward>(a, t, s, what);
    case kOpAf4H: return pick_rows<kOpAf4H, kLinForward>(a, t, s, what);
    default: return pick_rows<kOpAf8H, kLinForward>(a, t, s, what);
  }
}

}  // namespace mgq
