// Shared by the kernels of the matrix products (linear*.hip): the arguments,
// the operand types, the lookup of an output tile's group, MFMA calls and the
// epilogue.
//
// Every product is out[q][p] = sum_c Q[q][c] P[p][c] for one group:
//   forward  q = list entry, p = weight row (out feature), c = in feature;
//   dgrad    q = list entry, p = in feature,  c = weight row;
//   wgrad    q = weight row, p = in feature,  c = list entry of the group.
// p is the output's contiguous dimension. P feeds the MFMA's A operand, so a
// lane ends up with four consecutive p of one q (an 8-byte store of 16-bit
// results). An operand is "plain" when its contraction dimension is the
// contiguous one in memory (both operands of the forward product, dY in dgrad)
// and "transposed" otherwise (W in dgrad, both operands of wgrad).
#pragma once

#include "mgq_capi.h"
#include "mgq_common.h"

namespace mgq {

// Operand types. The MX forms are the weight's; their other operand is bf16.
enum LinOp : int { kOpBF16 = 0, kOpF16 = 1, kOpI8 = 2, kOpMx4 = 3, kOpMx8 = 4 };

struct LinArgs {
  const char* P;         // weight (forward, dgrad) or X (wgrad)
  const char* Q;         // X (forward) or dY
  const uint8_t* Ps;     // E8M0 scale bytes of an MX weight [G, np, nc / 32]
  int64_t ldp, ldq;      // row pitches in bytes
  int64_t p_group;       // bytes from one group's weight to the next
  const int32_t* offsets;    // [G + 1], or null: one group of all entries
  const int32_t* row_index;  // [M], or null: entry t reads row t
  int64_t M;             // list entries
  int64_t n_rows;        // rows of the gathered operand
  int G;
  int np, nq, nc;        // nq: wgrad only; nc: forward and dgrad only
  char* out;
  int64_t ldo;           // elements
  int64_t o_group;       // wgrad: elements from one group's output to the next
  int out_type;          // DType
  const float* sx;       // int8: scale of each X row
  const float* sw;       // int8: scale of each weight row [G, np]
  const float* bias;     // int8: [G, np] or null
};

typedef __bf16 lin_bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 lin_bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 lin_f16x8_t __attribute__((ext_vector_type(8)));
typedef float lin_f32x16_t __attribute__((ext_vector_type(16)));
typedef float lin_f32x4_t __attribute__((ext_vector_type(4)));
typedef int lin_i32x16_t __attribute__((ext_vector_type(16)));
typedef int lin_i32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t lin_u32x4_t __attribute__((ext_vector_type(4)));

// 16 bytes at an address aligned to one element only.
struct __attribute__((packed, aligned(1))) lin_u128_u_t {
  uint32_t v[4];
};

template <int OP>
constexpr bool lin_is_mx() {
  return OP == kOpMx4 || OP == kOpMx8;
}
// Bytes of one element of the Q operand (and of a dense P operand).
template <int OP>
constexpr int lin_esize() {
  return OP == kOpI8 ? 1 : 2;
}

template <int OP>
struct LinAcc {
  typedef lin_f32x16_t t32;  // a 32x32 block
  typedef lin_f32x4_t t16;   // a 16x16 block
};
template <>
struct LinAcc<kOpI8> {
  typedef lin_i32x16_t t32;
  typedef lin_i32x4_t t16;
};

// One MFMA over 16 bytes of each operand's row per lane: K = 16 (16-bit) or 32
// (int8) for the 32x32 block, twice that for the 16x16 block.
template <int OP>
__device__ __forceinline__ typename LinAcc<OP>::t32 lin_mfma32(lin_u32x4_t a, lin_u32x4_t b,
                                                               typename LinAcc<OP>::t32 c) {
  if constexpr (OP == kOpI8)
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(lin_i32x4_t, a),
                                                 __builtin_bit_cast(lin_i32x4_t, b), c, 0, 0, 0);
  else if constexpr (OP == kOpF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lin_f16x8_t, a),
                                                  __builtin_bit_cast(lin_f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf16x8_t, a),
                                                   __builtin_bit_cast(lin_bf16x8_t, b), c, 0, 0,
                                                   0);
}

// Eight MX codes and their group's scale byte -> eight bf16. The code's value
// (2 or 4 significant bits) times a power of two is exact in bf16 down to its
// subnormal step 2^-133. The conversion reads the scale's exponent field only,
// so byte 0 (2^-127) needs no care.
__device__ __forceinline__ lin_u32x4_t lin_decode_mx4(uint32_t codes, uint32_t scale_byte) {
  const float s = u2f(scale_byte << 23);
  lin_u32x4_t r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, 3));
  return r;
}
__device__ __forceinline__ lin_u32x4_t lin_decode_mx8(uint32_t lo, uint32_t hi,
                                                      uint32_t scale_byte) {
  const float s = u2f(scale_byte << 23);
  lin_u32x4_t r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true));
  return r;
}

// ---------------------------------------------------------------------------
// Which tile a workgroup computes. The offsets stay on the device (no host
// sync), so the grid is the host's bound on the tile count and every workgroup
// finds its tile itself; those past the count end at once.
//
// The list entries fall into G + 2 segments: the groups', and the entries
// before offsets[0] and from offsets[G] on, which belong to no group and get
// zeros. Offsets are clamped to [0, M], so that no entry outside the list is
// touched whatever they hold.
// ---------------------------------------------------------------------------
struct LinTile {
  int g;          // group; >= G: entries of no group
  int pt;         // tile along p
  int q0;         // first list entry
  int q_end;      // end of the segment
};

__device__ __forceinline__ int64_t lin_offset(const LinArgs& a, int i) {
  const int64_t v = a.offsets[i];
  return v < 0 ? 0 : (v > a.M ? a.M : v);
}

__device__ __forceinline__ void lin_segment(const LinArgs& a, int seg, int64_t* b, int64_t* e) {
  if (seg < a.G) {
    *b = lin_offset(a, seg);
    *e = lin_offset(a, seg + 1);
  } else if (seg == a.G) {
    *b = lin_offset(a, a.G);
    *e = a.M;
  } else {
    *b = 0;
    *e = seg == a.G + 1 ? lin_offset(a, 0) : 0;
  }
}

// Sum of v over this lane and the lanes below it: four DPP shifts inside the
// rows of 16 lanes, then the rows' last lanes broadcast to the rows above.
__device__ __forceinline__ uint32_t lin_wave_scan(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Every wave of the workgroup calls this with the same arguments. BM list
// entries per tile, n_pt tiles along p. Workgroups are dealt to the eight XCDs
// round robin, so workgroup b takes tile (b % 8) * (total / 8) + b / 8 of the
// list: an XCD's concurrent tiles are neighbours and share rows in its L2.
// Inside a group the tiles go in strips along q, p outer: the 32 tiles that an XCD
// runs at a time are then 8 along q and 4 along p, or all of p and 32 / n_pt along q
// where that is less, so that a row of Q is fetched once.
//
// A lane holds the bounds of up to kSegRegs segments, all loaded at once: a
// single token's product takes a few microseconds, of which every dependent load
// here would be a tenth. More segments than 64 kSegRegs are read in a loop, twice.
constexpr int kSegRegs = 4;
template <int BM>
__device__ inline bool lin_find_tile(const LinArgs& a, uint32_t n_pt, LinTile* t) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t bid = blockIdx.x;
  auto tiles_of = [](int64_t b, int64_t e) -> uint32_t {
    return e > b ? static_cast<uint32_t>(static_cast<uint64_t>(e - b + BM - 1) / BM) : 0u;
  };
  auto remap = [&](uint32_t total) -> uint32_t {
    const uint32_t x = bid & 7, rem = total & 7;
    return x * (total >> 3) + (x < rem ? x : rem) + (bid >> 3);
  };
  uint32_t id, base = 0, tiles = 0;
  int32_t b = 0, e = static_cast<int32_t>(a.M);
  int g = 0;
  if (!a.offsets) {
    tiles = tiles_of(0, a.M);
    if (bid >= tiles * n_pt) return false;
    id = remap(tiles * n_pt);
  } else if (a.G + 2 <= 64 * kSegRegs) {
    int32_t sb[kSegRegs], se[kSegRegs];
    uint32_t own[kSegRegs], incl[kSegRegs];
#pragma unroll
    for (int k = 0; k < kSegRegs; ++k) {
      const int s = 64 * k + static_cast<int>(lane);
      sb[k] = a.offsets[s <= a.G ? s : a.G];
      se[k] = a.offsets[s < a.G ? s + 1 : 0];
    }
    uint32_t total = 0;
#pragma unroll
    for (int k = 0; k < kSegRegs; ++k) {
      // segment s: offsets[s] to offsets[s + 1], with M after the last one; then
      // the entries before the first
      const int s = 64 * k + static_cast<int>(lane);
      sb[k] = s <= a.G ? sb[k] : 0;
      se[k] = s == a.G ? e : (s <= a.G + 1 ? se[k] : 0);
      sb[k] = sb[k] < 0 ? 0 : (sb[k] > e ? e : sb[k]);
      se[k] = se[k] < 0 ? 0 : (se[k] > e ? e : se[k]);
      own[k] = se[k] > sb[k] ? static_cast<uint32_t>(se[k] - sb[k] + BM - 1) / BM : 0u;
      incl[k] = total + lin_wave_scan(own[k]);
      total = __builtin_amdgcn_readlane(incl[k], 63);
    }
    if (bid >= total * n_pt) return false;
    id = remap(total * n_pt);
    const uint32_t mt = id / n_pt;
    bool found = false;
#pragma unroll
    for (int k = 0; k < kSegRegs; ++k) {
      const uint64_t hit = __ballot(mt >= incl[k] - own[k] && mt < incl[k]);
      if (!found && hit) {
        const int src = __builtin_ctzll(hit);
        found = true;
        g = 64 * k + src;
        tiles = __builtin_amdgcn_readlane(own[k], src);
        base = __builtin_amdgcn_readlane(incl[k], src) - tiles;
        b = __builtin_amdgcn_readlane(sb[k], src);
        e = __builtin_amdgcn_readlane(se[k], src);
      }
    }
    if (!found) return false;  // offsets that overlap may wrap the sums
  } else {
    uint32_t total = 0;
    for (int s0 = 0; s0 < a.G + 2; s0 += 64) {
      int64_t lo = 0, hi = 0;
      if (s0 + static_cast<int>(lane) < a.G + 2) lin_segment(a, s0 + lane, &lo, &hi);
      total += __builtin_amdgcn_readlane(lin_wave_scan(tiles_of(lo, hi)), 63);
    }
    if (bid >= total * n_pt) return false;
    id = remap(total * n_pt);
    const uint32_t mt = id / n_pt;
    bool found = false;
    for (int s0 = 0; s0 < a.G + 2 && !found; s0 += 64) {
      int64_t lo = 0, hi = 0;
      if (s0 + static_cast<int>(lane) < a.G + 2) lin_segment(a, s0 + lane, &lo, &hi);
      const uint32_t own = tiles_of(lo, hi), incl = base + lin_wave_scan(own);
      const uint64_t hit = __ballot(mt >= incl - own && mt < incl);
      if (hit) {
        const int src = __builtin_ctzll(hit);
        found = true;
        g = s0 + src;
        tiles = __builtin_amdgcn_readlane(own, src);
        base = __builtin_amdgcn_readlane(incl, src) - tiles;
        b = __builtin_amdgcn_readlane(static_cast<int32_t>(lo), src);
        e = __builtin_amdgcn_readlane(static_cast<int32_t>(hi), src);
      } else {
        base = __builtin_amdgcn_readlane(incl, 63);
      }
    }
    if (!found) return false;
  }
  const uint32_t local = id - base * n_pt;
  const uint32_t wide = n_pt > 8 || n_pt < 4 ? 8 : 32 / n_pt;
  const uint32_t strip = local / (wide * n_pt);
  const uint32_t in = local - strip * wide * n_pt;
  const uint32_t left = tiles - strip * wide;
  const uint32_t sm = left < wide ? left : wide;
  t->g = __builtin_amdgcn_readfirstlane(g);
  t->pt = __builtin_amdgcn_readfirstlane(static_cast<int>(in / sm));
  t->q0 = __builtin_amdgcn_readfirstlane(b + static_cast<int>((strip * wide + in % sm) * BM));
  t->q_end = __builtin_amdgcn_readfirstlane(e);
  return true;
}

// Row of the gathered operand that list entry t reads (indexes are clamped,
// never followed out of the matrix).
__device__ __forceinline__ int64_t lin_row(const LinArgs& a, int64_t t) {
  int64_t r = t;
  if (a.row_index) r = a.row_index[t];
  r = r < 0 ? 0 : r;
  return r < a.n_rows ? r : a.n_rows - 1;
}

// ---------------------------------------------------------------------------
// Epilogue: four consecutive p of one q, rounded once to the output type.
// ---------------------------------------------------------------------------
// Elements p .. p + 3 of an fp32 row of np (the last one again past its end).
__device__ __forceinline__ void lin_load4(const float* row, int p, int np, float (&v)[4]) {
  if (p + 4 <= np) {
    const f32x4_u_t f = load_f32x4(row + p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = row[p + i < np ? p + i : np - 1];
  }
}

// int8: (acc * sx) * sw + b, in fp32; the int32 sum is rounded to fp32 first.
template <int OP>
__device__ __forceinline__ void lin_scale4(const LinArgs& a, int g, int p, float sx, float (&v)[4]) {
  if constexpr (OP == kOpI8) {
    const int64_t c = static_cast<int64_t>(g) * a.np;
    float w[4], b[4] = {0, 0, 0, 0};
    lin_load4(a.sw + c, p, a.np, w);
    if (a.bias) lin_load4(a.bias + c, p, a.np, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = v[i] * sx * w[i];
      if (a.bias) v[i] = v[i] + b[i];
    }
  }
}

// Two results rounded half-even to 16 bits (one conversion each pair on bf16).
template <int TYPE>
__device__ __forceinline__ uint32_t lin_pack2(float x, float y) {
  if constexpr (TYPE == kF16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(x), static_cast<_Float16>(y)});
  } else {
    return __builtin_bit_cast(uint32_t,
                              lin_bf16x2_t{static_cast<__bf16>(x), static_cast<__bf16>(y)});
  }
}
__device__ __forceinline__ uint16_t lin_round16(float v, int type) {
  return type == kF16 ? f32_to_f16_rne(v) : f32_to_bf16_rne(v);
}

// row: the output row's first element; p: first column. Four results leave in one
// store at any address (a row of odd length starts anywhere).
struct __attribute__((packed, aligned(2))) lin_u64_u_t {
  uint32_t v[2];
};
__device__ __forceinline__ void lin_store4(const LinArgs& a, char* row, int p, const float (&v)[4]) {
  if (a.out_type == kF32) {
    float* o = reinterpret_cast<float*>(row) + p;
    if (p + 4 <= a.np) {
      *reinterpret_cast<f32x4_u_t*>(o) = f32x4_u_t{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p + i < a.np) o[i] = v[i];
    }
    return;
  }
  uint16_t* o = reinterpret_cast<uint16_t*>(row) + p;
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = lin_round16(v[i], a.out_type);
  if (p + 4 <= a.np) {
    lin_u64_u_t u;
    u.v[0] = h[0] | (static_cast<uint32_t>(h[1]) << 16);
    u.v[1] = h[2] | (static_cast<uint32_t>(h[3]) << 16);
    *reinterpret_cast<lin_u64_u_t*>(o) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < a.np) o[i] = h[i];
  }
}

}  // namespace mgq
