// The inner product that the kernels for a handful of rows share (affine_few.h,
// experts_up.hip, experts_down.hip): up to 16 NQ rows of 16-bit x times 16 NP weight rows in any
// of the weight formats, over a part of the contraction.
//
// A 16x16x32 MFMA takes the x rows as its A operand and the weight rows as B, so a
// lane ends up with four x rows (4 quad + e) of ONE weight row (lane % 16), and what
// belongs to a weight row (its scales, its bias) is one number a lane.
//
// A step is 128 elements of the contraction, four MFMAs. Lane (r, quad) reads what it
// needs of weight row r straight from memory:
//   dense       four 16-byte pieces, elements 32 j + 8 quad of the step for MFMA j;
//   MXFP        the 32 codes of the step's group `quad` and their scale byte, decoded
//               to bf16 exactly; MFMA j takes codes 8 j .. 8 j + 7 of every group;
//   affine      the 32 codes of the step's block `quad`. Since w = q s + b,
//                 sum_k x w = s sum_k x q + b sum_k x      over the ks of one group,
//               and q is exact in 16 bits: the MFMAs multiply with q itself, another
//               one with ones gives sum x in the same layout, and s and b are applied
//               in fp32 once for each block of 32 (of 64 for longer groups). For that an
//               MFMA has to stay inside a block: a 4 x 4 transposition among the quads
//               (permlane swaps) hands MFMA j the codes of block j.
// Scales come through LDS, 16 groups of a row at a time: a load of the two bytes that a
// step needs of each of 16 rows costs as much as the step's codes (a 14336 x 4096 weight of
// 4 bits times 16 rows: 22 us with such loads, 14 without any).
// Up to four x rows (NE = 1) sit at A rows 0, 4, 8, 12, so that only one of a lane's
// four results counts and s and b are applied to that one alone.
#pragma once

#include "linear_common.h"

namespace mgq {

enum FewFormat : int { kFewDense = 0, kFewMx4 = 1, kFewMx8 = 2, kFewAf2 = 3, kFewAf4 = 4, kFewAf8 = 5 };

constexpr int kFewStep = 128;

// A weight [groups, N, K] in its format.
struct FewWeight {
  const char* p;       // elements or codes
  const char* s;       // MXFP: E8M0 bytes [groups, N, K / 32]; affine: scales [groups, N, K >> shift]
  const char* b;       // affine: biases
  int64_t ld, group;   // bytes from row to row, from group to group
  int64_t n;           // rows of a group
  int shift;           // affine: log2 of the values that share a scale
  int type;            // affine: DType of scales and biases
};

// Bytes of a weight row at most: a lane's offset from the first of sixteen rows is 32 bits.
constexpr int64_t kFewRowBytes = int64_t(1) << 28;

// W: FewFormat, XT: kBF16 or kF16, SB: bytes of an affine scale (2 or 4).
template <int W_, int XT_, int SB_ = 2>
struct FewFmt {
  static constexpr int W = W_, XT = XT_, SB = SB_;
  static constexpr bool dense = W == kFewDense;
  static constexpr bool mx = W == kFewMx4 || W == kFewMx8;
  static constexpr bool affine = W >= kFewAf2;
  static constexpr int bits = dense ? 16 : W == kFewAf2 ? 2 : W == kFewMx4 || W == kFewAf4 ? 4 : 8;
  static constexpr int words = dense ? 16 : bits;  // 32-bit words of a lane and step
};

// Where a lane reads weight row p0 + lane % 16 (the last one of the weight past its end):
// addresses that are the same in all lanes, and the lane's offsets from them.
struct FewRow {
  const char* p;
  const char* s;
  const char* b;
  uint32_t lp, ls;
};

template <class F>
__device__ __forceinline__ FewRow few_row(const FewWeight& w, int64_t g, int p0, int K) {
  const uint32_t r16 = threadIdx.x & 15, quad = (threadIdx.x >> 4) & 3;
  const uint32_t left = static_cast<uint32_t>(w.n) - 1 - p0, r = r16 < left ? r16 : left;
  FewRow row;
  row.p = w.p + g * w.group + p0 * w.ld;
  row.lp = r * static_cast<uint32_t>(w.ld) + quad * (F::dense ? 16 : 4 * F::bits);
  row.s = row.b = nullptr;
  row.ls = 0;
  if constexpr (!F::dense) {
    const uint32_t n = F::mx ? K / 32 : K >> w.shift;
    const int64_t at = (g * w.n + p0) * n * (F::mx ? 1 : F::SB);
    row.s = w.s + at;
    row.ls = r * n * (F::mx ? 1 : F::SB);
    if constexpr (F::affine) row.b = w.b + at;
  }
  return row;
}

// What a lane holds of a step.
template <class F>
struct FewStep {
  uint32_t v[F::words];
};

struct __attribute__((packed, aligned(4))) few_u64_u_t {
  uint32_t v[2];
};

// 16 bytes at any address.
__device__ __forceinline__ lin_u32x4_t few_load16(const char* at) {
  const lin_u128_u_t u = *reinterpret_cast<const lin_u128_u_t*>(at);
  return lin_u32x4_t{u.v[0], u.v[1], u.v[2], u.v[3]};
}
// Elements k .. k + 7 of a 16-bit row of K, zeros from K on.
__device__ __forceinline__ lin_u32x4_t few_cut16(const char* row, int k, int K) {
  lin_u32x4_t r = {0, 0, 0, 0};
  if (k + 8 <= K) return few_load16(row + 2 * static_cast<int64_t>(k));
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < K)
      r[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k + i]) << (16 * (i & 1));
  return r;
}

template <int BYTES>
__device__ __forceinline__ uint32_t few_param(const char* at) {
  if constexpr (BYTES == 2) return *reinterpret_cast<const uint16_t*>(at);
  return *reinterpret_cast<const uint32_t*>(at);
}

// Step s of a weight row. WHOLE: the row holds all 128 elements of it; otherwise zeros
// follow the row's end (dense), or a block past it reads the row's first one and
// few_multiply discards it (quantized, K % 32 == 0).
template <class F, bool WHOLE>
__device__ __forceinline__ void few_load(FewStep<F>& f, const FewRow& r, int s, int K) {
  const uint32_t quad = (threadIdx.x >> 4) & 3;
  if constexpr (F::dense) {
    const uint32_t at = r.lp + static_cast<uint32_t>(s) * (2 * kFewStep);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lin_u32x4_t u;
      if constexpr (WHOLE)
        u = few_load16(r.p + static_cast<uint64_t>(at + 64 * j));
      else
        u = few_cut16(r.p + static_cast<uint64_t>(r.lp) - 16 * quad, s * kFewStep + 32 * j + 8 * quad, K);
#pragma unroll
      for (int i = 0; i < 4; ++i) f.v[4 * j + i] = u[i];
    }
  } else {
    uint32_t at = r.lp + static_cast<uint32_t>(s) * (16 * F::bits);
    if constexpr (!WHOLE) {
      const bool inside = s * kFewStep + 32 * quad < static_cast<uint32_t>(K);
      at = inside ? at : r.lp - quad * (4 * F::bits);
    }
    const char* from = r.p + static_cast<uint64_t>(at);
    if constexpr (F::bits == 2) {
      const few_u64_u_t u = *reinterpret_cast<const few_u64_u_t*>(from);
      f.v[0] = u.v[0];
      f.v[1] = u.v[1];
    } else {
#pragma unroll
      for (int h = 0; h < F::bits / 4; ++h) {
        const lin_u32x4_t u = few_load16(from + 16 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) f.v[4 * h + i] = u[i];
      }
    }
  }
}

// A lane's x elements of a step's MFMAs. `row` is the lane's x row.
template <class F, bool WHOLE>
__device__ __forceinline__ void few_load_x(lin_u32x4_t (&x)[4], const char* row, int s, int K) {
  const int quad = (threadIdx.x >> 4) & 3;
  const int k0 = s * kFewStep + (F::mx ? 32 : 8) * quad;
  constexpr int step = F::mx ? 8 : 32;
  const char* at = row + 2 * static_cast<int64_t>(k0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (WHOLE)
      x[j] = few_load16(at + 2 * step * j);
    else if constexpr (F::dense)
      x[j] = few_cut16(row, k0 + step * j, K);
    else  // (whole pieces: K % 32 == 0)
      x[j] = k0 + step * j < K ? few_load16(at + 2 * step * j) : lin_u32x4_t{0, 0, 0, 0};
  }
}

template <class F>
__device__ __forceinline__ lin_f32x4_t few_mfma(lin_u32x4_t x, lin_u32x4_t w, lin_f32x4_t c) {
  if constexpr (F::XT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lin_f16x8_t, x),
                                                  __builtin_bit_cast(lin_f16x8_t, w), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lin_bf16x8_t, x),
                                                   __builtin_bit_cast(lin_bf16x8_t, w), c, 0, 0, 0);
}

// Word q of quad i, for word i of quad q: the 4 x 4 transposition among the quads.
__device__ __forceinline__ void few_transpose(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  const auto u = __builtin_amdgcn_permlane32_swap(a, c, false, false);
  const auto v = __builtin_amdgcn_permlane32_swap(b, d, false, false);
  const auto p = __builtin_amdgcn_permlane16_swap(u[0], v[0], false, false);
  const auto q = __builtin_amdgcn_permlane16_swap(u[1], v[1], false, false);
  a = p[0];
  b = p[1];
  c = q[0];
  d = q[1];
}

// Four codes (one a byte, below 16) as two pairs of 16-bit numbers. A byte below 16 is
// the E4M3 number byte * 2^-9 (subnormals below 8, the first binade from 8 on), so the
// scaled conversion of two E4M3 numbers returns the integers.
template <int XT>
__device__ __forceinline__ void few_small(uint32_t bytes, uint32_t& lo, uint32_t& hi) {
  if constexpr (XT == kF16) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.0f, true));
  } else {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.0f, true));
  }
}
// Four 8-bit codes: whole numbers up to 255 are exact in both types.
template <int XT>
__device__ __forceinline__ void few_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = lin_pack2<XT>(static_cast<float>(w & 0xff), static_cast<float>((w >> 8) & 0xff));
  hi = lin_pack2<XT>(static_cast<float>((w >> 16) & 0xff), static_cast<float>(w >> 24));
}

// The codes of an affine step after the transposition, ready to be decoded: eight codes
// of block j for every lane, in the order of k = 32 j + 8 quad + 0..7.
template <class F>
__device__ __forceinline__ void few_arrange(FewStep<F>& f) {
  if constexpr (F::bits == 4) {
    few_transpose(f.v[0], f.v[1], f.v[2], f.v[3]);
  } else if constexpr (F::bits == 8) {
    few_transpose(f.v[0], f.v[2], f.v[4], f.v[6]);
    few_transpose(f.v[1], f.v[3], f.v[5], f.v[7]);
  }
}
template <class F>
__device__ __forceinline__ lin_u32x4_t few_codes(const FewStep<F>& f, const uint32_t (&half)[4], int j) {
  lin_u32x4_t r;
  uint32_t a, b, c, d;
  if constexpr (F::bits == 4) {
    const uint32_t even = f.v[j] & 0x0f0f0f0fu, odd = (f.v[j] >> 4) & 0x0f0f0f0fu;
    few_small<F::XT>(__builtin_amdgcn_perm(odd, even, 0x05010400u), a, b);
    few_small<F::XT>(__builtin_amdgcn_perm(odd, even, 0x07030602u), c, d);
  } else if constexpr (F::bits == 8) {
    few_bytes<F::XT>(f.v[2 * j], a, b);
    few_bytes<F::XT>(f.v[2 * j + 1], c, d);
  } else {
    // eight 2-bit codes: two a byte, then as above
    const uint32_t n = (half[j] & 0xffu) | ((half[j] & 0xff00u) << 8);
    const uint32_t lo4 = (n & 0x000f000fu) | ((n & 0x00f000f0u) << 4);
    const uint32_t even = lo4 & 0x03030303u, odd = (lo4 >> 2) & 0x03030303u;
    few_small<F::XT>(__builtin_amdgcn_perm(odd, even, 0x05010400u), a, b);
    few_small<F::XT>(__builtin_amdgcn_perm(odd, even, 0x07030602u), c, d);
  }
  r[0] = a;
  r[1] = b;
  r[2] = c;
  r[3] = d;
  return r;
}

// Scales of 16 groups of a wave's weight rows in LDS, the wave's own: affine (s, b) as two
// floats, MXFP the bytes. A lane brings four groups of its row from memory.
constexpr int kFewGroups = 16;
template <class F>
constexpr int few_pitch() {  // bytes of a row
  return F::mx ? kFewGroups + 4 : 8 * (kFewGroups + 1);
}
template <class F, int NP>
constexpr int few_lds() {  // bytes of a wave
  return F::dense ? 0 : NP * 16 * few_pitch<F>();
}
template <class F>
struct FewParams {
  uint32_t s[F::affine ? F::SB : 1], b[F::affine ? F::SB : 1];  // four groups
};
template <int B>
struct __attribute__((packed, aligned(B))) few_params_u_t {
  uint32_t v[B];
};
// Four values of B bytes from g on of a row of n, those past its end like its last.
template <int B>
__device__ __forceinline__ void few_fetch4(const char* row, int g, int n, uint32_t (&v)[B]) {
  if (g + 4 <= n) {
    const few_params_u_t<B> u =
        *reinterpret_cast<const few_params_u_t<B>*>(row + static_cast<uint64_t>(g) * B);
#pragma unroll
    for (int i = 0; i < B; ++i) v[i] = u.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < B; ++i) v[i] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* at = row + static_cast<uint64_t>(g + i < n ? g + i : n - 1) * B;
      if constexpr (B == 1)
        v[0] |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t*>(at)) << (8 * i);
      else if constexpr (B == 2)
        v[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at)) << (16 * (i & 1));
      else
        v[i] = *reinterpret_cast<const uint32_t*>(at);
    }
  }
}
template <class F>
__device__ __forceinline__ void few_fetch(FewParams<F>& f, const FewRow& r, int g0, int n) {
  const int g = g0 + 4 * static_cast<int>((threadIdx.x >> 4) & 3);
  few_fetch4<F::affine ? F::SB : 1>(r.s + static_cast<uint64_t>(r.ls), g, n, f.s);
  if constexpr (F::affine) few_fetch4<F::SB>(r.b + static_cast<uint64_t>(r.ls), g, n, f.b);
}
template <int SB>
__device__ __forceinline__ uint32_t few_param_f32(uint32_t raw, int type) {
  if constexpr (SB == 4) return raw;
  return type == kF16 ? f2u(f16_to_f32(static_cast<uint16_t>(raw))) : raw << 16;
}
// Into LDS (the wave's reads of what was there are done: LDS serves a wave in order; the
// fences keep the compiler to that).
template <class F, int NP>
__device__ __forceinline__ void few_stage(const FewParams<F> (&f)[NP], int type, char* lds) {
  const int r16 = threadIdx.x & 15, quad = (threadIdx.x >> 4) & 3;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  auto put = [&](auto as_f32) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      char* row = lds + (16 * p + r16) * few_pitch<F>();
      if constexpr (F::mx) {
        *reinterpret_cast<uint32_t*>(row + 4 * quad) = f[p].s[0];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t s = F::SB == 4 ? f[p].s[i] : f[p].s[i / 2] >> (16 * (i & 1)) & 0xffff;
          const uint32_t b = F::SB == 4 ? f[p].b[i] : f[p].b[i / 2] >> (16 * (i & 1)) & 0xffff;
          *reinterpret_cast<uint2*>(row + 8 * (4 * quad + i)) = uint2{as_f32(s), as_f32(b)};
        }
      }
    }
  };
  // (one branch on the type, not one a value)
  if (F::SB == 2 && type == kF16)
    put([](uint32_t v) { return f2u(f16_to_f32(static_cast<uint16_t>(v))); });
  else
    put([](uint32_t v) { return F::SB == 2 ? v << 16 : v; });
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// acc[p][q] += the step's product of weight rows p with x rows q. `first`: the group of
// element 0 of the step, counted from the first one in LDS.
template <class F, int NP, int NQ, int NE, bool WHOLE>
__device__ __forceinline__ void few_multiply(FewStep<F> (&f)[NP], const lin_u32x4_t (&x)[NQ][4], int s,
                                             int K, int shift, int first, const char* lds,
                                             lin_f32x4_t (&acc)[NP][NQ]) {
  const int r16 = threadIdx.x & 15, quad = (threadIdx.x >> 4) & 3;
  if constexpr (F::dense) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const lin_u32x4_t w = {f[p].v[4 * j], f[p].v[4 * j + 1], f[p].v[4 * j + 2], f[p].v[4 * j + 3]};
#pragma unroll
        for (int q = 0; q < NQ; ++q) acc[p][q] = few_mfma<F>(x[q][j], w, acc[p][q]);
      }
  } else if constexpr (F::mx) {
    uint32_t scale[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p)
      scale[p] = *reinterpret_cast<const uint8_t*>(lds + (16 * p + r16) * few_pitch<F>() + first + quad);
    if constexpr (!WHOLE) {  // (x is zero there, but a code may stand for no number)
      const uint32_t keep = s * kFewStep + 32 * quad < K ? 0xffffffffu : 0u;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
#pragma unroll
        for (int i = 0; i < F::words; ++i) f[p].v[i] &= keep;
        scale[p] &= keep;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        lin_u32x4_t w;
        if constexpr (F::W == kFewMx4)
          w = lin_decode_mx4(f[p].v[j], scale[p]);
        else
          w = lin_decode_mx8(f[p].v[2 * j], f[p].v[2 * j + 1], scale[p]);
#pragma unroll
        for (int q = 0; q < NQ; ++q) acc[p][q] = few_mfma<F>(x[q][j], w, acc[p][q]);
      }
  } else {
    const uint32_t one = F::XT == kF16 ? 0x3c003c00u : 0x3f803f80u;
    const lin_u32x4_t ones = {one, one, one, one};
    const lin_f32x4_t zero = {0, 0, 0, 0};
    uint32_t half[NP][4];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      few_arrange<F>(f[p]);
      if constexpr (F::bits == 2) {
        // 16 codes a word, words 0 and 1 of block `quad`: MFMA j's quads 0 and 1 take
        // the halves of word 0 of block j, quads 2 and 3 those of word 1
        const auto u = __builtin_amdgcn_permlane32_swap(f[p].v[0], f[p].v[1], false, false);
        const auto a = __builtin_amdgcn_permlane16_swap(u[0], u[0], false, false);
        const auto b = __builtin_amdgcn_permlane16_swap(u[1], u[1], false, false);
        const uint32_t up = 16 * (quad & 1);
        half[p][0] = (a[0] >> up) & 0xffffu;
        half[p][1] = (a[1] >> up) & 0xffffu;
        half[p][2] = (b[0] >> up) & 0xffffu;
        half[p][3] = (b[1] >> up) & 0xffffu;
      }
    }
    // blocks j .. j + N - 1 lie in one group
    auto blocks = [&](int j, auto n) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value;
      lin_f32x4_t sum[NQ];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        sum[q] = few_mfma<F>(x[q][j], ones, zero);
        if constexpr (N == 2) sum[q] = few_mfma<F>(x[q][j + 1], ones, sum[q]);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const float2 sb = *reinterpret_cast<const float2*>(
            lds + (16 * p + r16) * few_pitch<F>() + 8 * (first + (32 * j >> shift)));
        const lin_u32x4_t w0 = few_codes<F>(f[p], half[p], j);
        lin_u32x4_t w1;
        if constexpr (N == 2) w1 = few_codes<F>(f[p], half[p], j + 1);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          lin_f32x4_t d = few_mfma<F>(x[q][j], w0, zero);
          if constexpr (N == 2) d = few_mfma<F>(x[q][j + 1], w1, d);
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            acc[p][q][e] = fmaf(sb.x, d[e], acc[p][q][e]);
            acc[p][q][e] = fmaf(sb.y, sum[q][e], acc[p][q][e]);
          }
        }
      }
    };
    if (WHOLE && shift > 5) {
      blocks(0, std::integral_constant<int, 2>{});
      blocks(2, std::integral_constant<int, 2>{});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!WHOLE && s * kFewStep + 32 * j >= K) break;
        blocks(j, std::integral_constant<int, 1>{});
      }
    }
  }
}

// Steps [s_begin, s_end) of NP weight rows (a lane's own) with NQ x rows. The operands of
// DEPTH - 1 steps are in flight beyond the one being multiplied: x too, whose trip from L2
// would otherwise be waited for in every step. A step that the rows end in comes last, by
// itself. lds: few_lds<F, NP>() bytes of the wave's own.
template <class F, int NP, int NQ, int NE, int DEPTH>
__device__ __forceinline__ void few_product(const FewRow (&row)[NP], const FewWeight& w,
                                            const char* const (&x)[NQ], int K, int s_begin, int s_end,
                                            char* lds, lin_f32x4_t (&acc)[NP][NQ]) {
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int q = 0; q < NQ; ++q) acc[p][q] = lin_f32x4_t{0, 0, 0, 0};
  if (s_begin >= s_end) return;
  const int whole = K / kFewStep, end = s_end < whole ? s_end : whole;
  const int shift = F::affine ? w.shift : 5, groups = K >> shift;
  const int period = (kFewGroups << shift) / kFewStep;  // steps of the groups in LDS
  int group = s_begin * kFewStep >> shift;              // the first one there
  FewParams<F> par[NP];
  auto fetch = [&](int g) __attribute__((always_inline)) {
    if constexpr (!F::dense) {
#pragma unroll
      for (int p = 0; p < NP; ++p) few_fetch<F>(par[p], row[p], g, groups);
    }
  };
  // before step s: its groups into LDS, the next ones on their way
  auto stage = [&](int s) __attribute__((always_inline)) {
    if constexpr (!F::dense) {
      if (((s - s_begin) & (period - 1)) == 0) {
        few_stage<F, NP>(par, w.type, lds);
        group = s * kFewStep >> shift;
        if (s + period < s_end) fetch((s + period) * kFewStep >> shift);
      }
    }
  };
  FewStep<F> f[DEPTH][NP];
  lin_u32x4_t xv[DEPTH][NQ][4];
  auto load = [&](int d, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < NP; ++p) few_load<F, true>(f[d][p], row[p], s, K);
#pragma unroll
    for (int q = 0; q < NQ; ++q) few_load_x<F, true>(xv[d][q], x[q], s, K);
  };
  fetch(group);
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d)
    if (s_begin + d < end) load(d, s_begin + d);
  for (int s = s_begin; s < end; s += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (s + d >= end) break;
      if (s + d + DEPTH - 1 < end) load((d + DEPTH - 1) % DEPTH, s + d + DEPTH - 1);
      stage(s + d);
      few_multiply<F, NP, NQ, NE, true>(f[d], xv[d], s + d, K, shift,
                                        ((s + d) * kFewStep >> shift) - group, lds, acc);
    }
  }
  if (s_end > whole) {
#pragma unroll
    for (int p = 0; p < NP; ++p) few_load<F, false>(f[0][p], row[p], whole, K);
#pragma unroll
    for (int q = 0; q < NQ; ++q) few_load_x<F, false>(xv[0][q], x[q], whole, K);
    stage(whole);
    few_multiply<F, NP, NQ, NE, false>(f[0], xv[0], whole, K, shift, (whole * kFewStep >> shift) - group,
                                       lds, acc);
  }
}

}  // namespace mgq
