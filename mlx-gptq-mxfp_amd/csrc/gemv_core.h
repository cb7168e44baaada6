// One row of x times many weight rows in any of few_core.h's formats, for single tokens.
//
// L lanes (64, 32 or 16) share a weight row, 16 bytes (8 for 2-bit codes) each, so that a
// load instruction reads 64 / L rows in contiguous pieces of up to 1 KB: 5.3 TB/s of cold
// weight measured against 4.4 where sixteen rows are read 64 bytes at a time, as an MFMA
// operand wants them, both by loads alone. With the products the kernels reach 4.3 to 4.5 TB/s
// of bf16 and 3.1 of 4-bit codes, launch included, whose two waves a SIMD (174 registers) keep
// less in flight. A lane multiplies its codes with the x values beside them (two
// products an instruction, fp32 sums); scales and biases apply to the lane's sum, since its
// codes lie in one group. The lanes' sums of a row are added once, at the end.
#pragma once

#include "few_core.h"

namespace mgq {

template <class F>
constexpr int gemv_elems() {  // of a lane's piece
  return F::dense ? 8 : F::bits == 8 ? 16 : 32;
}
template <class F>
constexpr int gemv_words() {
  return gemv_elems<F>() * F::bits / 32;
}

// 16-bit pairs times pairs, added to c.
template <int XT>
__device__ __forceinline__ float gemv_dot2(uint32_t a, uint32_t b, float c) {
  if constexpr (XT == kF16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
  } else {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(lin_bf16x2_t, a),
                                           __builtin_bit_cast(lin_bf16x2_t, b), c, false);
  }
}

// A piece of one load instruction's rows, and of x (pairs; sum: of the piece).
template <class F>
struct GemvPiece {
  uint32_t v[gemv_words<F>()];
  uint32_t s, b;
};
template <class F>
struct GemvX {
  uint32_t v[gemv_elems<F>() / 2];
  float sum;
};

// Pairs in the order in which gemv_multiply decodes: (0 2)(4 6)(1 3)(5 7) of every eight
// for 2- and 4-bit affine codes, as they lie for the others.
template <class F>
__device__ __forceinline__ void gemv_arrange(GemvX<F>& x) {
  constexpr int N = gemv_elems<F>() / 2;
  if constexpr (F::affine) {
    const uint32_t one = F::XT == kF16 ? 0x3c003c00u : 0x3f803f80u;
    float sum = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) sum = gemv_dot2<F::XT>(x.v[i], one, sum);
    x.sum = sum;
  }
  if constexpr (F::affine && F::bits < 8) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint32_t a = x.v[i], b = x.v[i + 1], c = x.v[i + 2], d = x.v[i + 3];
      x.v[i] = __builtin_amdgcn_perm(b, a, 0x05040100u);
      x.v[i + 1] = __builtin_amdgcn_perm(d, c, 0x05040100u);
      x.v[i + 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      x.v[i + 3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
    }
  }
}

// Eight 4-bit E2M1 numbers times 2 as four pairs.
template <int XT>
__device__ __forceinline__ lin_u32x4_t gemv_pairs(uint32_t v) {
  lin_u32x4_t r;
  if constexpr (XT == kF16) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 2.0f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 2.0f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 2.0f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 2.0f, 3));
  } else {
    r = lin_decode_mx4(v, 128);
  }
  return r;
}

// The piece's product with x, the sum of its XS parts.
template <class F, int XS>
__device__ __forceinline__ float gemv_multiply(const GemvPiece<F>& f, const GemvX<F> (&x)[XS], int type) {
  float r = 0;
  auto add = [&](uint32_t w, int pair) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < XS; ++i) r = gemv_dot2<F::XT>(w, x[i].v[pair], r);
  };
  if constexpr (F::dense) {
#pragma unroll
    for (int i = 0; i < 4; ++i) add(f.v[i], i);
  } else if constexpr (F::mx) {
#pragma unroll
    for (int i = 0; i < gemv_words<F>(); i += F::W == kFewMx8 ? 2 : 1) {
      lin_u32x4_t w;
      if constexpr (F::W == kFewMx4)
        w = lin_decode_mx4(f.v[i], f.s);
      else
        w = lin_decode_mx8(f.v[i], f.v[i + 1], f.s);
      const int at = F::W == kFewMx4 ? 4 * i : 2 * i;
#pragma unroll
      for (int j = 0; j < 4; ++j) add(w[j], at + j);
    }
  } else {
    if constexpr (F::bits == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t lo, hi;
        few_bytes<F::XT>(f.v[i], lo, hi);
        add(lo, 2 * i);
        add(hi, 2 * i + 1);
      }
    } else if constexpr (F::bits == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t p[4];
        few_small<F::XT>(f.v[i] & 0x0f0f0f0fu, p[0], p[1]);
        few_small<F::XT>((f.v[i] >> 4) & 0x0f0f0f0fu, p[2], p[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) add(p[j], 4 * i + j);
      }
    } else {
      // a 2-bit code in four bits is the E2M1 number code / 2
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t even = f.v[i] & 0x33333333u, odd = (f.v[i] >> 2) & 0x33333333u;
        const lin_u32x4_t e = gemv_pairs<F::XT>(even), o = gemv_pairs<F::XT>(odd);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          add(e[2 * j], 8 * i + 4 * j);
          add(e[2 * j + 1], 8 * i + 4 * j + 1);
          add(o[2 * j], 8 * i + 4 * j + 2);
          add(o[2 * j + 1], 8 * i + 4 * j + 3);
        }
      }
    }
    r = u2f(few_param_f32<F::SB>(f.s, type)) * r;
    float sum = x[0].sum;
#pragma unroll
    for (int i = 1; i < XS; ++i) sum += x[i].sum;
    r = fmaf(u2f(few_param_f32<F::SB>(f.b, type)), sum, r);
  }
  return r;
}

// acc[i] += (this lane's part of) weight rows first(i) + lane / L times x, over the chunks
// [c0, c1) of L pieces each; a row has gemv_chunks of them. first(i) is the same in all
// lanes and leaves 64 / L rows to the weight's end. x is the sum of XS rows of K, one after the
// other. The weights of DEPTH - 1 chunks are in flight beyond the one being multiplied.
template <class F, int L>
__host__ __device__ inline int gemv_chunks(int K) {
  constexpr int E = L * gemv_elems<F>();
  return (K + E - 1) / E;
}
template <class F, int L, int R, int DEPTH, int XS = 1, typename First>
__device__ __forceinline__ void gemv_add(float (&acc)[R], const FewWeight& w, int64_t g, First&& first,
                                         const char* x, int K, int c0, int c1) {
  constexpr int E = gemv_elems<F>();
  const int lane = threadIdx.x & 63;
  const uint32_t sub = lane / L;  // row of the instruction's rows
  GemvPiece<F> f[DEPTH][R];
  GemvX<F> xv[DEPTH][XS];
  auto load = [&](int d, int c) __attribute__((always_inline)) {
    const int k0 = (c * L + (lane & (L - 1))) * E;
    const bool whole = (c + 1) * L * E <= K;
    if constexpr (F::dense) {
      if (whole) {
#pragma unroll
        for (int p = 0; p < XS; ++p) {
          const lin_u32x4_t u = few_load16(x + 2 * (static_cast<int64_t>(p) * K + k0));
#pragma unroll
          for (int i = 0; i < 4; ++i) xv[d][p].v[i] = u[i];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const char* base = w.p + g * w.group + first(r) * w.ld;
          const lin_u32x4_t v = few_load16(base + static_cast<uint64_t>(sub * static_cast<uint32_t>(w.ld) + 2u * k0));
#pragma unroll
          for (int i = 0; i < 4; ++i) f[d][r].v[i] = v[i];
        }
      } else {
#pragma unroll
        for (int p = 0; p < XS; ++p) {
          const lin_u32x4_t u = few_cut16(x + 2 * static_cast<int64_t>(p) * K, k0, K);
#pragma unroll
          for (int i = 0; i < 4; ++i) xv[d][p].v[i] = u[i];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const lin_u32x4_t v = few_cut16(w.p + g * w.group + (first(r) + sub) * w.ld, k0, K);
#pragma unroll
          for (int i = 0; i < 4; ++i) f[d][r].v[i] = v[i];
        }
      }
    } else {
      const uint32_t kc = k0 < K ? k0 : 0;  // (a lane past the row's end reads its first piece)
#pragma unroll
      for (int p = 0; p < XS; ++p)
#pragma unroll
        for (int h = 0; h < E / 8; ++h) {
          const lin_u32x4_t u =
              few_load16(x + 2 * static_cast<int64_t>(p) * K + static_cast<uint64_t>(2u * kc + 16u * h));
#pragma unroll
          for (int i = 0; i < 4; ++i) xv[d][p].v[4 * h + i] = u[i];
        }
      const uint32_t at = sub * static_cast<uint32_t>(w.ld) + kc / 32 * (4 * F::bits) + kc % 32 * F::bits / 8;
      const int n = F::affine ? K >> w.shift : K / 32;  // scales of a row
      const uint32_t ps = (sub * n + (F::affine ? kc >> w.shift : kc / 32)) * (F::affine ? F::SB : 1);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = first(r);
        const char* base = w.p + g * w.group + row * w.ld;
        if constexpr (F::bits == 2) {
          const few_u64_u_t u = *reinterpret_cast<const few_u64_u_t*>(base + static_cast<uint64_t>(at));
          f[d][r].v[0] = u.v[0];
          f[d][r].v[1] = u.v[1];
        } else {
          const lin_u32x4_t u = few_load16(base + static_cast<uint64_t>(at));
#pragma unroll
          for (int i = 0; i < 4; ++i) f[d][r].v[i] = u[i];
        }
        const int64_t srow = (g * w.n + row) * n;
        if constexpr (F::mx) {
          f[d][r].s = *reinterpret_cast<const uint8_t*>(w.s + srow + static_cast<uint64_t>(ps));
        } else {
          f[d][r].s = few_param<F::SB>(w.s + srow * F::SB + static_cast<uint64_t>(ps));
          f[d][r].b = few_param<F::SB>(w.b + srow * F::SB + static_cast<uint64_t>(ps));
        }
      }
    }
  };
  auto multiply = [&](int d, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < XS; ++p) gemv_arrange<F>(xv[d][p]);
    const bool inside = F::dense || (c * L + (lane & (L - 1))) * E < K;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float v = gemv_multiply<F, XS>(f[d][r], xv[d], w.type);
      acc[r] += inside ? v : 0.0f;
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d)
    if (c0 + d < c1) load(d, c0 + d);
  for (int c = c0; c < c1; c += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (c + d >= c1) break;
      if (c + d + DEPTH - 1 < c1) load((d + DEPTH - 1) % DEPTH, c + d + DEPTH - 1);
      multiply(d, c + d);
    }
  }
}

// Sums over the lanes of a row. Afterwards sum[q], in all lanes of the wave's quarter i
// (16 lanes), is row gemv_row<L>(q, i) of the wave's R 64 / L rows (row r of them: load r /
// (64 / L), lanes r % (64 / L)).
template <int L, int R>
constexpr int gemv_sums() {
  return R * 16 / L;
}
template <int L>
__device__ __forceinline__ int gemv_row(int q, int quarter) {
  return 4 * q + (L == 16 ? quarter : (quarter & 1) * 2 + (quarter >> 1));
}
template <int L, int R>
__device__ __forceinline__ void gemv_reduce(const float (&acc)[R], float (&sum)[gemv_sums<L, R>()]) {
  constexpr int N = gemv_sums<L, R>();
  float half[2 * N];
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) {
    if constexpr (L == 64) {
      const auto s = __builtin_amdgcn_permlane32_swap(f2u(acc[2 * i]), f2u(acc[2 * i + 1]), false, false);
      half[i] = u2f(s[0]) + u2f(s[1]);
    } else if constexpr (L == 32) {
      half[i] = acc[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v;
    if constexpr (L == 16) {
      v = acc[i];
    } else {
      const auto s = __builtin_amdgcn_permlane16_swap(f2u(half[2 * i]), f2u(half[2 * i + 1]), false, false);
      v = u2f(s[0]) + u2f(s[1]);
    }
    auto ror = [](float x, auto n) {
      return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x),
                                                                   0x120 + n, 0xf, 0xf, true));
    };
    v += ror(v, std::integral_constant<int, 8>{});
    v += ror(v, std::integral_constant<int, 4>{});
    v += ror(v, std::integral_constant<int, 2>{});
    sum[i] = v + ror(v, std::integral_constant<int, 1>{});
  }
}

// Lanes of a row for a contraction of K: the fewest idle ones, the longest pieces among
// about equal counts. Rows of the weight that one load instruction takes must exist.
template <class F>
inline int gemv_lanes(int64_t K, int64_t rows) {
  const int64_t pieces = ceil_div(K, gemv_elems<F>());
  int best = 64;
  for (int l = 32; l >= 16; l /= 2)
    if (64 / l <= rows && 10 * ceil_div(pieces, l) * l < 9 * ceil_div(pieces, best) * best) best = l;
  return best;
}

}  // namespace mgq
