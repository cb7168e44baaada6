// Products with affine weights, y[t, n] = sum_k x[r(t), k] (q[g, n, k] s + b) with a scale
// s and a bias b for each group of 32, 64 or 128 values of a weight row and 2-, 4- or
// 8-bit codes q, packed low bits first. The list of entries t and its groups g are those of
// linear_common.h, the arithmetic is few_core.h's.
//
// Few rows: a workgroup computes 16 NQ entries (4 where NE = 1) x 16 NP weight rows; its
// waves share the contraction and add their sums through LDS in wave order.
#include "gemv_core.h"
#include "linear_few.h"

namespace mgq {
namespace {

template <class F, int NP, int NQ, int NE, int WAVES, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES) affine_few_kernel(const LinArgs a, const FewWeight w) {
  constexpr int BM = NE == 1 ? 4 : 16 * NQ;
  __shared__ lin_f32x4_t part[WAVES * NP * NQ * 64];
  __shared__ __attribute__((aligned(16))) char params[WAVES * few_lds<F, NP>()];
  LinTile t;
  if (!lin_find_tile<BM>(a, (a.np + 16 * NP - 1) / (16 * NP), &t)) return;
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = t.pt * 16 * NP;
  const int steps = t.g < a.G ? (a.nc + kFewStep - 1) / kFewStep : 0;  // (no group: zeros)
  const int64_t g = t.g < a.G ? t.g : 0;

  FewRow row[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i)
    row[i] = few_row<F>(w, g, p0 + 16 * i < a.np ? p0 + 16 * i : p0, a.nc);
  const char* x[NQ];
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    const int64_t q = t.q0 + (NE == 1 ? r16 >> 2 : 16 * j + r16);
    x[j] = a.Q + lin_row(a, q < t.q_end ? q : t.q_end - 1) * a.ldq;
  }
  lin_f32x4_t acc[NP][NQ];
  few_product<F, NP, NQ, NE, DEPTH>(row, w, x, a.nc, steps * wave / WAVES, steps * (wave + 1) / WAVES,
                                    params + wave * few_lds<F, NP>(), acc);
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) part[((wave * NP + i) * NQ + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int blk = wave; blk < NP * NQ; blk += WAVES) {
    lin_f32x4_t sum = part[blk * 64 + lane];
#pragma unroll
    for (int o = 1; o < WAVES; ++o) {
      const lin_f32x4_t v = part[(o * NP * NQ + blk) * 64 + lane];
#pragma unroll
      for (int e = 0; e < NE; ++e) sum[e] += v[e];
    }
    const int p = p0 + 16 * (blk / NQ) + r16;
    if (p >= a.np) continue;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int64_t q = t.q0 + (NE == 1 ? quad : 16 * (blk % NQ) + 4 * quad + e);
      if (q < t.q_end)
        reinterpret_cast<uint16_t*>(a.out)[q * a.ldo + p] = lin_round16(sum[e], a.out_type);
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

template <class F, int NP, int NQ, int NE, int WAVES, int DEPTH>
int launch_few(const LinArgs& a, const FewWeight& w, hipStream_t s, const char* what) {
  const int64_t grid = lin_row_tiles(a, NE == 1 ? 4 : 16 * NQ) * ceil_div(a.np, 16 * NP);
  MGQ_REQUIRE(grid < kLinFewGrid * 4 / WAVES, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  affine_few_kernel<F, NP, NQ, NE, WAVES, DEPTH>
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
#ifdef AFFINE_FORCE
extern "C" int mgq_force[4] = {0, 0, 0, 0};
#endif

template <class F>
int run(const LinArgs& a, const FewWeight& w, hipStream_t s, const char* what) {
#ifdef AFFINE_FORCE
  const int per = mgq_force[1];
  switch (mgq_force[0]) {
    case 5: return launch_gemv<F>(a, w, s, what);
    case 1: return launch_few<F, 1, 1, 1, 4, 4>(a, w, s, what);
    case 2: return launch_few<F, 2, 1, 1, 4, 4>(a, w, s, what);
    case 3: return launch_few<F, 4, 1, 1, 4, 4>(a, w, s, what);
    case 6: return launch_few<F, 1, 1, 4, 4, 4>(a, w, s, what);
    case 7: return launch_few<F, 2, 1, 4, 4, 2>(a, w, s, what);
    case 8: return launch_few<F, 2, 1, 4, 4, 4>(a, w, s, what);
    case 9: return launch_few<F, 4, 1, 4, 4, 2>(a, w, s, what);
    case 10: return launch_few<F, 4, 1, 4, 4, 4>(a, w, s, what);
    case 11: return launch_few<F, 4, 1, 4, 8, 2>(a, w, s, what);
    case 12: return launch_few<F, 4, 1, 4, 8, 4>(a, w, s, what);
    case 13: return launch_few<F, 4, 2, 4, 4, 2>(a, w, s, what);
    case 14: return launch_few<F, 4, 2, 4, 4, 3>(a, w, s, what);
    case 15: return launch_few<F, 4, 4, 4, 4, 2>(a, w, s, what);
    case 16: return launch_few<F, 2, 4, 4, 4, 2>(a, w, s, what);
    case 30: case 31: case 32: case 33: {
      LinArgs b = a;
      b.P = w.p; b.Ps = reinterpret_cast<const uint8_t*>(w.s); b.Pb = reinterpret_cast<const uint8_t*>(w.b);
      b.ldp = w.ld; b.p_group = w.group; b.p_shift = w.shift; b.p_type = w.type;
      const int op = (F::XT == kF16 ? kOpAf2H : kOpAf2) + (F::W - kFewAf2);
      const int r[4] = {256, 128, 64, 64}, c[4] = {256, 256, 256, 128};
      const int i = mgq_force[0] - 30;
      return lin_tile_affine(b, op, LinTileShape{r[i], c[i], mgq_force[2] != 0}, s, what);
    }
  }
#endif
  if (a.M <= 4) return launch_few<F, 1, 1, 1, 4, 2>(a, w, s, what);
  if (a.M <= 16 || (a.offsets && a.M <= 16 * static_cast<int64_t>(a.G)))
    return launch_few<F, 1, 1, 4, 4, 2>(a, w, s, what);
  return launch_few<F, 2, 4, 4, 4, 1>(a, w, s, what);
}
template <int XT, int SB>
int run_bits(int bits, const LinArgs& a, const FewWeight& w, hipStream_t s, const char* what) {
#ifdef AFFINE_FORCE
  return bits == 8 ? run<FewFmt<kFewAf8, kBF16, 2>>(a, w, s, what) : run<FewFmt<kFewAf4, kBF16, 2>>(a, w, s, what);
#endif
  if (bits == 2) return run<FewFmt<kFewAf2, XT, SB>>(a, w, s, what);
  if (bits == 4) return run<FewFmt<kFewAf4, XT, SB>>(a, w, s, what);
  return run<FewFmt<kFewAf8, XT, SB>>(a, w, s, what);
}

}  // namespace
}  // namespace mgq

using namespace mgq;

extern "C" int mgq_affine_linear(const void* X, int dtype, int64_t n_rows, int64_t ldx,
                                 const int32_t* row_index, int64_t n_entries, const uint32_t* words,
                                 const void* scales, const void* biases, int param_dtype, int bits,
                                 int64_t group_size, int64_t n_groups, int64_t N, int64_t K,
                                 const int32_t* offsets, void* Y, void* stream) {
  clear_error();
  const char* what = "affine_linear";
  MGQ_REQUIRE(dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE, "%s: bfloat16 or float16 rows only",
              what);
  MGQ_REQUIRE(param_dtype == kF32 || param_dtype == kBF16 || param_dtype == kF16, MGQ_ERR_VALUE,
              "%s: scales and biases are float32, bfloat16 or float16", what);
  MGQ_REQUIRE(bits == 2 || bits == 4 || bits == 8, MGQ_ERR_VALUE, "%s: bits must be 2, 4 or 8", what);
  MGQ_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128, MGQ_ERR_VALUE,
              "%s: group_size must be 32, 64 or 128", what);
  if (int rc = lin_check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(K % group_size == 0, MGQ_ERR_SHAPE, "%s: K = %lld is no multiple of the group size", what,
              (long long)K);
  MGQ_REQUIRE(ldx >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  if (n_entries == 0) return MGQ_OK;
  LinArgs a = {};
  a.Q = static_cast<const char*>(X);
  a.ldq = 2 * ldx;
  a.offsets = offsets;
  a.row_index = row_index;
  a.M = n_entries;
  a.n_rows = n_rows;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(N);
  a.nc = static_cast<int>(K);
  a.out = static_cast<char*>(Y);
  a.ldo = N;
  a.out_type = dtype;
  FewWeight w = {};
  w.p = reinterpret_cast<const char*>(words);
  w.s = static_cast<const char*>(scales);
  w.b = static_cast<const char*>(biases);
  w.ld = K / 8 * bits;
  w.group = w.ld * N;
  w.n = N;
  w.shift = group_size == 32 ? 5 : group_size == 64 ? 6 : 7;
  w.type = param_dtype;
  hipStream_t s = as_stream(stream);
  if (dtype == kF16)
    return param_dtype == kF32 ? run_bits<kF16, 4>(bits, a, w, s, what)
                               : run_bits<kF16, 2>(bits, a, w, s, what);
  return param_dtype == kF32 ? run_bits<kBF16, 4>(bits, a, w, s, what)
                             : run_bits<kBF16, 2>(bits, a, w, s, what);
}
