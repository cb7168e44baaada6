// The kernels of the product with affine weights for few rows (affine_linear.hip chooses
// among them), for one number of bits: affine_bits2.hip, affine_bits4.hip, affine_bits8.hip.
//
// affine_few_kernel: a workgroup computes 16 NQ entries (4 where NE = 1) x 16 NP weight rows a
// row block. Its waves are KS along the contraction, whose sums are added through LDS in wave
// order, times row blocks.
// affine_gemv_kernel: single entries (gemv_core.h).
//
// Bound by waits with few waves a SIMD. 128 experts of 1536 x 2048, 4 bits, 512 entries take
// 72 us (228 MB, 3.2 TB/s), of which the 17.6 million vector instructions (about 160 for a
// step of 128 values times 32 rows) are 29 at four cycles on 1024 SIMDs; its waves, three to a
// SIMD at 148 registers, wait for 55 % of their cycles. With cached weights it takes 63, so
// most of the wait is not memory's; more than one step in flight beyond the one that is
// multiplied took the same time. 14336 x 4096, 4 bits, one entry: 10.5 us (33 MB, 3.1 TB/s),
// 3.3 of them vector instructions.
#pragma once

#include "affine_few_choice.h"
#include "gemv_core.h"
#include "linear_few.h"

namespace mgq {
namespace {

template <class F, int NP, int NQ, int NE, int WAVES, int KS, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES) affine_few_kernel(const LinArgs a, const FewWeight w) {
  constexpr int BM = NE == 1 ? 4 : 16 * NQ, WR = WAVES / KS, BP = 16 * NP * WR;
  __shared__ lin_f32x4_t part[KS > 1 ? WAVES * NP * NQ * 64 : 1];
  __shared__ __attribute__((aligned(16))) char params[WAVES * few_lds<F, NP>()];
  LinTile t;
  if (!lin_find_tile<BM>(a, (a.np + BP - 1) / BP, &t)) return;
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % KS, rw = wave / KS;
  const int p0 = t.pt * BP + rw * 16 * NP;
  const int steps = t.g < a.G ? (a.nc + kFewStep - 1) / kFewStep : 0;  // (no group: zeros)
  const int64_t g = t.g < a.G ? t.g : 0;

  FewRow row[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i)  // (blocks past the weight's end repeat a row of it)
    row[i] = few_row<F>(w, g, p0 + 16 * i < a.np ? p0 + 16 * i : a.np - 1, a.nc);
  const char* x[NQ];
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    const int64_t q = t.q0 + (NE == 1 ? r16 >> 2 : 16 * j + r16);
    x[j] = a.Q + lin_row(a, q < t.q_end ? q : t.q_end - 1) * a.ldq;
  }
  lin_f32x4_t acc[NP][NQ];
  few_product<F, NP, NQ, NE, DEPTH>(row, w, x, a.nc, steps * kw / KS, steps * (kw + 1) / KS,
                                    params + wave * few_lds<F, NP>(), acc);
  auto store = [&](int i, int j, const lin_f32x4_t& v) {
    const int p = p0 + 16 * i + r16;
    if (p >= a.np) return;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int64_t q = t.q0 + (NE == 1 ? quad : 16 * j + 4 * quad + e);
      if (q < t.q_end)
        reinterpret_cast<uint16_t*>(a.out)[q * a.ldo + p] = lin_round16(v[e], a.out_type);
    }
  };
  if constexpr (KS == 1) {
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < NQ; ++j) store(i, j, acc[i][j]);
  } else {
    // the KS waves of a row block, in their order
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < NQ; ++j) part[((wave * NP + i) * NQ + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int blk = kw; blk < NP * NQ; blk += KS) {
      const lin_f32x4_t* from = part + (rw * KS * NP * NQ + blk) * 64 + lane;
      lin_f32x4_t sum = *from;
#pragma unroll
      for (int o = 1; o < KS; ++o) {
        const lin_f32x4_t v = from[o * NP * NQ * 64];
#pragma unroll
        for (int e = 0; e < NE; ++e) sum[e] += v[e];
      }
      store(blk / NQ, blk % NQ, sum);
    }
  }
}

// Single entries: a wave takes one entry and R 64 / L weight rows.
template <class F, int L, int R>
__global__ void __launch_bounds__(256) affine_gemv_kernel(const LinArgs a, const FewWeight w) {
  constexpr int RI = 64 / L, ROWS = R * RI;  // rows of a load, of a wave
  LinTile t;
  if (!lin_find_tile<1>(a, (a.np + 4 * ROWS - 1) / (4 * ROWS), &t)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = (4 * t.pt + wave) * ROWS;
  if (p0 >= a.np) return;
  auto first = [&](int r) { return p0 + r * RI < a.np - RI ? p0 + r * RI : a.np - RI; };
  float acc[R], sum[gemv_sums<L, R>()];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.0f;
  if (t.g < a.G)  // (no group: zeros)
    gemv_add<F, L, R, 2>(acc, w, t.g, first, a.Q + lin_row(a, t.q0) * a.ldq, a.nc, 0,
                         gemv_chunks<F, L>(a.nc));
  gemv_reduce<L, R>(acc, sum);
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + t.q0 * a.ldo;
#pragma unroll
  for (int q = 0; q < gemv_sums<L, R>(); ++q)
    if ((lane & 15) == q) {
      const int r = gemv_row<L>(q, lane >> 4);
      out[first(r / RI) + r % RI] = lin_round16(sum[q], a.out_type);
    }
}

template <class F, int NP, int NQ, int NE, int WAVES, int KS, int DEPTH>
int launch_few(const LinArgs& a, const FewWeight& w, hipStream_t s, const char* what) {
  const int64_t grid = lin_row_tiles(a, NE == 1 ? 4 : 16 * NQ) * ceil_div(a.np, 16 * NP * (WAVES / KS));
  MGQ_REQUIRE(grid < kLinFewGrid * 4 / WAVES, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  affine_few_kernel<F, NP, NQ, NE, WAVES, KS, DEPTH>
      <<<static_cast<unsigned>(grid), 64 * WAVES, 0, s>>>(a, w);
  return check_launch(what);
}
template <class F>
int launch_gemv(const LinArgs& a, const FewWeight& w, hipStream_t s, const char* what) {
  constexpr int R = 8;
  const int lanes = gemv_lanes<F>(a.nc, a.np);
  const int64_t grid = a.M * ceil_div(a.np, 4 * R * (64 / lanes));
  MGQ_REQUIRE(grid < kLinFewGrid, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  const unsigned blocks = static_cast<unsigned>(grid);
  if (lanes == 64) affine_gemv_kernel<F, 64, R><<<blocks, 256, 0, s>>>(a, w);
  else if (lanes == 32) affine_gemv_kernel<F, 32, R><<<blocks, 256, 0, s>>>(a, w);
  else affine_gemv_kernel<F, 16, R><<<blocks, 256, 0, s>>>(a, w);
  return check_launch(what);
}

template <class F>
int run(const LinArgs& a, const FewWeight& w, int choice, hipStream_t s, const char* what) {
  switch (choice) {
#define MGQ_CASE(n, np, nq, ne, waves, ks, depth, alone, shared) \
  case n: return launch_few<F, np, nq, ne, waves, ks, depth>(a, w, s, what);
    MGQ_AFFINE_SHAPES(MGQ_CASE)
#undef MGQ_CASE
    default: return launch_gemv<F>(a, w, s, what);
  }
}
template <int FORMAT>
int run_types(const LinArgs& a, const FewWeight& w, int choice, hipStream_t s, const char* what) {
  const bool f16 = a.out_type == kF16, wide = w.type == kF32;
  if (f16) return wide ? run<FewFmt<FORMAT, kF16, 4>>(a, w, choice, s, what)
                       : run<FewFmt<FORMAT, kF16, 2>>(a, w, choice, s, what);
  return wide ? run<FewFmt<FORMAT, kBF16, 4>>(a, w, choice, s, what)
              : run<FewFmt<FORMAT, kBF16, 2>>(a, w, choice, s, what);
}

}  // namespace
}  // namespace mgq
