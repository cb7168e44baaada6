// A routed layer's experts for a few rows, in two launches (experts_up.hip and
// experts_down.hip):
//
//   act[i] = silu(Wg[e] x[t]) * (Wu[e] x[t])          for entry i = t k + j, e = index[i]
//   out[t] = sum_j weights[t, j] Wd[e] act[t k + j]
//
// Entries whose expert is outside [0, E) add nothing.
#pragma once

#include "gemv_core.h"

namespace mgq {

constexpr int kDecodeRows = 64;     // rows of a call
constexpr int kDecodeTopK = 16;     // experts of a row
constexpr int kDecodeEntries = kDecodeRows * kDecodeTopK;
// Rows of a call up to which the activation goes from one launch to the other as the sum of
// two 16-bit numbers: itself rounded, and what that lost, rounded (2^-17 of it is lost in bf16,
// 2^-22 in f16, where one number loses about what rounding the result does). The second
// product's MFMA has rows to spare for them as long as an expert has at most 8 of the call's
// 64. Above, one number: an MFMA for each part makes 16 rows of 4-bit codes 45.4 us instead of
// 42.4 and 64 rows of MXFP8 192 instead of 177 (128 experts of 768 x 2048); experts cut into
// eights of their rows instead take 47.5 and 184.
constexpr int kDecodePartRows = 8;

struct DecodeArgs {
  const char* x;
  int64_t ldx;           // bytes
  const void* index;     // [T, k] int32 or int64
  const float* weights;  // [T, k]
  FewWeight up, down;    // [E, 2 I, H] (gate rows first), [E, H, I]
  uint16_t* act;         // workspace: [T k, act_parts, I] of x's type
  int32_t* plan;         // workspace: see decode_plan (experts_up.hip)
  int32_t* counts;       // workspace: parts of a column tile that are done
  float* sums;           // workspace: [parts, T, H]
  uint16_t* out;         // [T, H]
  int index64;
  int T, k, n;           // n = T k
  int E, H, I;
  int type;              // kBF16 or kF16
  int act_parts;         // 2 up to kDecodePartRows rows
  int parts, tiles;      // of the second launch
};

// The plan that the first launch leaves for the second one (T > 1): plan[0] items,
// then the items, then the entries. An item is one expert with up to kDecodeItem of its
// rows; entries of an item are (entry of act, weight as bits), each row once.
struct DecodeItem {
  int32_t expert;
  uint16_t first, count;
};
struct DecodeEntry {
  int32_t entry;
  float weight;
};
constexpr int kDecodeItem = 16;
constexpr int kDecodePlanHead = 16;  // bytes

// The second launch: 32 columns of the result a workgroup, whose items `decode_parts`
// workgroups share; what each gives goes through the workspace.
constexpr int kDecodeCols = 32;
inline int decode_tiles(int64_t H) { return static_cast<int>((H + kDecodeCols - 1) / kDecodeCols); }
inline int decode_parts(int64_t n, int64_t H) {
  const int64_t fill = 512 / decode_tiles(H), most = n / 8;  // two workgroups a CU, two items a wave
  const int64_t p = fill < most ? fill : most;
  return static_cast<int>(p < 1 ? 1 : p > 8 ? 8 : p);
}
inline int64_t decode_round(int64_t bytes) { return (bytes + 255) / 256 * 256; }
inline int decode_act_parts(int64_t T) { return T <= kDecodePartRows ? 2 : 1; }
inline int64_t decode_act_bytes(int64_t T, int64_t k, int64_t I) {
  return decode_round(T * k * decode_act_parts(T) * I * 2);
}
inline int64_t decode_plan_bytes(int64_t n) { return decode_round(kDecodePlanHead + n * 16); }
inline int64_t decode_count_bytes(int64_t H) { return decode_round(4 * int64_t(decode_tiles(H))); }

// The activation of entry `i` at p (an infinity, or no number, in one part).
__device__ __forceinline__ void decode_store_act(const DecodeArgs& a, int i, int p, float v) {
  const uint16_t high = lin_round16(v, a.type);
  uint16_t* row = a.act + static_cast<int64_t>(i) * a.act_parts * a.I + p;
  row[0] = high;
  if (a.act_parts == 1) return;
  const float left = v - (a.type == kF16 ? f16_to_f32(high) : bf16_to_f32(high));
  row[a.I] = fabsf(left) < INFINITY ? lin_round16(left, a.type) : 0;
}

__device__ __forceinline__ int decode_expert(const DecodeArgs& a, int i) {
  if (a.index64) {
    const int64_t e = static_cast<const int64_t*>(a.index)[i];
    return e >= 0 && e < a.E ? static_cast<int>(e) : -1;
  }
  const int32_t e = static_cast<const int32_t*>(a.index)[i];
  return e >= 0 && e < a.E ? e : -1;
}

int decode_up(const DecodeArgs& a, int format, hipStream_t s, const char* what);
int decode_down(const DecodeArgs& a, int format, hipStream_t s, const char* what);

// f(FewFmt) for a weight's format, the rows' type and the scales' size.
template <typename Fn>
int decode_dispatch(int format, int type, int param_type, Fn&& f) {
  const bool wide = param_type == kF32;
#define MGQ_AFFINE(FMT)                                        \
  if (type == kF16) {                                          \
    if (wide) return f(FewFmt<FMT, kF16, 4>{});                \
    return f(FewFmt<FMT, kF16, 2>{});                          \
  }                                                            \
  if (wide) return f(FewFmt<FMT, kBF16, 4>{});                 \
  return f(FewFmt<FMT, kBF16, 2>{});
  switch (format) {
    case kFewDense:
      if (type == kF16) return f(FewFmt<kFewDense, kF16>{});
      return f(FewFmt<kFewDense, kBF16>{});
    case kFewMx4: return f(FewFmt<kFewMx4, kBF16>{});
    case kFewMx8: return f(FewFmt<kFewMx8, kBF16>{});
    case kFewAf2: MGQ_AFFINE(kFewAf2)
    case kFewAf4: MGQ_AFFINE(kFewAf4)
    default: MGQ_AFFINE(kFewAf8)
  }
#undef MGQ_AFFINE
}

}  // namespace mgq
