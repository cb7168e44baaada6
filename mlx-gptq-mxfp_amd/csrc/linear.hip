// Matrix products grouped by expert: dense (bf16, f16), MXFP4 / MXFP8 and int8
// weights; both gradients of the dense form. Group g owns the list entries
// [offsets[g], offsets[g + 1]); entry t reads row row_index[t] of X (or row t).
//
// Here are the entry points: their checks, and which kernel takes a call.
#include <math.h>

#include "linear_few.h"

namespace mgq {
namespace {

// Which kernel and tile a product over rows takes: of those whose grid holds it, the
// one whose time by the model below is least. The model was fitted to 980 products (all
// types, 1 .. 16384 entries, 0 .. 128 groups, K 256 .. 14336, aligned and not) that were
// timed with each of their 3 to 7 choices, called again and again on the same weights, so
// that what fits the memory-side cache came from there. On these the model's choice costs
// 1.7 % over the best one on average and 64 % at worst, where the largest tile that the
// average group fills costs 33 % on average and tenfold at worst. (Pricing the few rows'
// weight at 2.86 TB/s had 46 % at worst, but sent one token through 8 experts to a tile,
// 16 instead of 11 us.) The worst are lists of some 3000 entries over 32 to 60 groups,
// whose tiles the model counts below the groups' number.
//
//   large tiles: rounds of the 256 CUs x (stages x time of a stage + a fixed time
//     for the tile's first loads and its results), or the weight's bytes at the
//     rate the tile's loads reach;
//   few rows: a wave's batches of loads one after the other, or the bytes that all
//     workgroups read through L2 (rows that a tile repeats are read once), or the
//     weight's bytes from memory at 4.35 TB/s. Loads off 16-byte boundaries cost 1.14
//     times as much, off 4-byte boundaries 2.7 times.
//
// How the entries fall into groups is not known here: each active group is taken
// to leave 0.58 tiles unfilled, and a tile of several entries to belong to a group
// 2.4 times as long as the average.
struct TileTime {
  int rows, cols;
  bool staged;
  double stage, fixed;  // us
};
constexpr TileTime kTileTimes[] = {
    {64, 128, false, 0.451, 2.2}, {64, 256, false, 0.483, 2.3}, {128, 256, false, 0.806, 2.6},
    {256, 256, false, 1.18, 3.2}, {64, 128, true, 0.581, 3.0}, {64, 256, true, 1.19, 3.2},
    {128, 256, true, 1.75, 3.2},
};

// A kernel of few rows (nq blocks of 16 entries) or a tile; neither where no kernel's
// grid holds the product.
struct RowsChoice {
  int nq;
  LinTileShape tile;
};

template <int OP, int KIND>
RowsChoice choose_rows(const LinArgs& a) {
  const bool direct = lin_tile_direct(a, OP, KIND);
  const int64_t es = lin_esize<OP>();
  const double wb = OP == kOpMx4 ? 0.53 : OP == kOpMx8 ? 1.03 : es;  // bytes of a weight
  const double M = static_cast<double>(a.M), np = a.np, nc = a.nc;
  const double active = a.offsets ? (a.G < a.M ? a.G : M) : 1;
  const double weight_bytes = active * np * nc * wb;
  auto row_tiles = [&](int rows) {
    return a.offsets ? fmax(1.0, M / rows + 0.575 * active) : ceil(M / rows);
  };
  double best = 1e300;
  RowsChoice choice = {};
  for (const TileTime& t : kTileTimes) {
    if (t.staged == direct || lin_tile_grid(a, t.rows, t.cols) >= kLinTileGrid) continue;
    double rounds = row_tiles(t.rows) * ceil(np / t.cols) / 256;
    rounds = rounds < 1 ? 1 : rounds + 0.617 * (ceil(rounds) - rounds);
    const double stage = t.stage * (wb < 1 ? 0.92 : 1.0);
    const double us = 2 + fmax(rounds * (ceil(nc * es / 128) * stage + t.fixed),
                               weight_bytes / (direct ? 12.5e6 : 8.1e6));
    if (us < best) {
      best = us;
      choice.tile = LinTileShape{t.rows, t.cols, t.staged};
    }
  }
  if (KIND == kLinForward) {
    const uintptr_t bounds = lin_row_bounds(a, a.nc * es);
    const double cost = (bounds & 3) ? 2.72 : (bounds & 15) ? 1.14 : 1.0;
    for (const int nq : {1, 2, 4}) {
      if (lin_few_grid(a, nq) >= kLinFewGrid) continue;
      const int rows = 16 * nq, cols = lin_few_cols(nq), batch = nq == 4 ? 4 : 8;
      const double read = fmin(rows, ceil(M / active * (a.offsets && M > active ? 2.44 : 1.0)));
      const double l2 = row_tiles(rows) * ceil(np / cols) * (cols * wb + read * es) * nc * cost;
      const double chain = ceil(ceil(nc * es / 256) / batch) * batch * (nq + cols / 16) * 0.125 * cost;
      const double us = 5.45 + fmax(chain, fmax(l2 / 6.25e6, weight_bytes / 4.35e6));
      if (us < best) {
        best = us;
        choice.nq = nq;
      }
    }
  }
  return choice;
}

template <int OP, int KIND>
int run_rows(const LinArgs& a, hipStream_t s, const char* what) {
  const RowsChoice c = choose_rows<OP, KIND>(a);
  MGQ_REQUIRE(c.nq || c.tile.rows, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  return c.nq ? lin_few_rows(a, OP, c.nq, s, what) : lin_tile_rows(a, OP, KIND, c.tile, s, what);
}

}  // namespace
}  // namespace mgq

using namespace mgq;

extern "C" int mgq_grouped_linear(const void* X, int dtype, int64_t n_rows, int64_t ldx,
                                  const int32_t* row_index, int64_t n_entries, const void* W,
                                  int64_t n_groups, int64_t N, int64_t K, int64_t ldw,
                                  int64_t w_group, const int32_t* offsets, void* Y, void* stream) {
  clear_error();
  const char* what = "grouped_linear";
  MGQ_REQUIRE(dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE, "%s: bfloat16 or float16 only", what);
  if (int rc = lin_check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(ldx >= K && ldw >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  if (n_entries == 0) return MGQ_OK;
  LinArgs a = {};
  a.P = static_cast<const char*>(W);
  a.Q = static_cast<const char*>(X);
  a.ldp = 2 * ldw;
  a.ldq = 2 * ldx;
  a.p_group = 2 * w_group;
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
  hipStream_t s = as_stream(stream);
  return dtype == kF16 ? run_rows<kOpF16, kLinForward>(a, s, what)
                       : run_rows<kOpBF16, kLinForward>(a, s, what);
}

extern "C" int mgq_grouped_dgrad(const void* dY, int dtype, int64_t n_entries, int64_t lddy,
                                 const void* W, int64_t n_groups, int64_t N, int64_t K, int64_t ldw,
                                 int64_t w_group, const int32_t* offsets, void* dX, int out_dtype,
                                 void* stream) {
  clear_error();
  const char* what = "grouped_dgrad";
  MGQ_REQUIRE(dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE, "%s: bfloat16 or float16 only", what);
  MGQ_REQUIRE(out_dtype == dtype || out_dtype == kF32, MGQ_ERR_VALUE,
              "%s: the result has the operands' type or float32", what);
  if (int rc = lin_check_list(what, offsets, nullptr, n_groups, n_entries, n_entries)) return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(lddy >= N && ldw >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  if (n_entries == 0 || K == 0) return MGQ_OK;
  LinArgs a = {};
  a.P = static_cast<const char*>(W);
  a.Q = static_cast<const char*>(dY);
  a.ldp = 2 * ldw;
  a.ldq = 2 * lddy;
  a.p_group = 2 * w_group;
  a.offsets = offsets;
  a.M = n_entries;
  a.n_rows = n_entries;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(K);
  a.nc = static_cast<int>(N);
  a.out = static_cast<char*>(dX);
  a.ldo = K;
  a.out_type = out_dtype;
  hipStream_t s = as_stream(stream);
  return dtype == kF16 ? run_rows<kOpF16, kLinDgrad>(a, s, what)
                       : run_rows<kOpBF16, kLinDgrad>(a, s, what);
}

extern "C" int64_t mgq_grouped_wgrad_workspace_size(int64_t n_entries, int64_t n_groups, int64_t N,
                                                    int64_t K) {
  if (n_entries < 0 || n_groups < 1 || N < 1 || K < 1) return 0;
  return lin_tile_wgrad_bytes(n_entries, n_groups, N, K);
}

extern "C" int mgq_grouped_wgrad(const void* dY, int dtype, int64_t n_entries, int64_t lddy,
                                 const void* X, int64_t n_rows, int64_t ldx,
                                 const int32_t* row_index, int64_t n_groups, int64_t N, int64_t K,
                                 const int32_t* offsets, void* dW, int out_dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* what = "grouped_wgrad";
  MGQ_REQUIRE(dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE, "%s: bfloat16 or float16 only", what);
  MGQ_REQUIRE(out_dtype == dtype || out_dtype == kF32, MGQ_ERR_VALUE,
              "%s: the result has the operands' type or float32", what);
  if (int rc = lin_check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(lddy >= N && ldx >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  MGQ_REQUIRE(n_groups <= kLinPlanGroups, MGQ_ERR_SHAPE, "%s: %lld groups (at most %d)", what,
              (long long)n_groups, kLinPlanGroups);
  const int64_t need = mgq_grouped_wgrad_workspace_size(n_entries, n_groups, N, K);
  MGQ_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), MGQ_ERR_WORKSPACE,
              "%s: workspace %lld < %lld bytes", what, (long long)workspace_bytes, (long long)need);
  if (K == 0) return MGQ_OK;
  LinArgs a = {};
  a.P = static_cast<const char*>(X);
  a.Q = static_cast<const char*>(dY);
  a.ldp = 2 * ldx;
  a.ldq = 2 * lddy;
  a.offsets = offsets;
  a.row_index = row_index;
  a.M = n_entries;
  a.n_rows = n_rows;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(K);
  a.nq = static_cast<int>(N);
  a.out = static_cast<char*>(dW);
  a.ldo = K;
  a.o_group = N * K;
  a.out_type = out_dtype;
  hipStream_t s = as_stream(stream);
  return lin_tile_wgrad(a, dtype == kF16 ? kOpF16 : kOpBF16, workspace, s, what);
}

extern "C" int mgq_mxfp_linear(const void* X, int64_t n_rows, int64_t ldx, const int32_t* row_index,
                               int64_t n_entries, const uint32_t* words, const uint8_t* scales,
                               int mode, int64_t n_groups, int64_t N, int64_t K,
                               const int32_t* offsets, void* Y, void* stream) {
  clear_error();
  const char* what = "mxfp_linear";
  MGQ_REQUIRE(mode == kMxfp4 || mode == kMxfp8, MGQ_ERR_VALUE, "%s: mode must be mxfp4 or mxfp8",
              what);
  if (int rc = lin_check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(K % kMxGroup == 0, MGQ_ERR_SHAPE, "%s: K = %lld is no multiple of 32", what,
              (long long)K);
  MGQ_REQUIRE(ldx >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  if (n_entries == 0) return MGQ_OK;
  LinArgs a = {};
  a.P = reinterpret_cast<const char*>(words);
  a.Q = static_cast<const char*>(X);
  a.Ps = scales;
  a.ldp = mode == kMxfp4 ? K / 2 : K;
  a.ldq = 2 * ldx;
  a.p_group = a.ldp * N;
  a.offsets = offsets;
  a.row_index = row_index;
  a.M = n_entries;
  a.n_rows = n_rows;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(N);
  a.nc = static_cast<int>(K);
  a.out = static_cast<char*>(Y);
  a.ldo = N;
  a.out_type = kBF16;
  hipStream_t s = as_stream(stream);
  return mode == kMxfp4 ? run_rows<kOpMx4, kLinForward>(a, s, what)
                        : run_rows<kOpMx8, kLinForward>(a, s, what);
}

extern "C" int mgq_int8_linear(const int8_t* X, const float* x_scale, int64_t n_rows, int64_t ldx,
                               const int32_t* row_index, int64_t n_entries, const int8_t* W,
                               const float* w_scale, const float* bias, int64_t n_groups, int64_t N,
                               int64_t K, int64_t ldw, int64_t w_group, const int32_t* offsets,
                               void* Y, int out_dtype, void* stream) {
  clear_error();
  const char* what = "int8_linear";
  MGQ_REQUIRE(out_dtype == kF32 || out_dtype == kBF16 || out_dtype == kF16, MGQ_ERR_VALUE,
              "%s: the result is float32, bfloat16 or float16", what);
  if (int rc = lin_check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  // |sum| <= 128 * 128 * K has to fit the int32 accumulator
  MGQ_REQUIRE(K <= 131071, MGQ_ERR_SHAPE, "%s: K = %lld exceeds 131071 (int32 sums)", what,
              (long long)K);
  MGQ_REQUIRE(ldx >= K && ldw >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  if (n_entries == 0) return MGQ_OK;
  LinArgs a = {};
  a.P = reinterpret_cast<const char*>(W);
  a.Q = reinterpret_cast<const char*>(X);
  a.ldp = ldw;
  a.ldq = ldx;
  a.p_group = w_group;
  a.offsets = offsets;
  a.row_index = row_index;
  a.M = n_entries;
  a.n_rows = n_rows;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(N);
  a.nc = static_cast<int>(K);
  a.out = static_cast<char*>(Y);
  a.ldo = N;
  a.out_type = out_dtype;
  a.sx = x_scale;
  a.sw = w_scale;
  a.bias = bias;
  return run_rows<kOpI8, kLinForward>(a, as_stream(stream), what);
}

extern "C" int mgq_linear_choice(int product, const void* X, int64_t ldx, int64_t n_entries,
                                 const void* W, int64_t n_groups, int64_t N, int64_t K, int64_t ldw,
                                 int64_t w_group, int grouped, int32_t* tile) {
  clear_error();
  const char* what = "linear_choice";
  MGQ_REQUIRE(product >= 0 && product <= 6, MGQ_ERR_VALUE, "%s: no such product", what);
  const int32_t some_list = 0;  // stands for offsets: the choice does not read them
  if (int rc = lin_check_list(what, grouped ? &some_list : nullptr, nullptr, n_groups, n_entries,
                              n_entries))
    return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  const bool dgrad = product >= 5, mx4 = product == kOpMx4, mx8 = product == kOpMx8;
  const int es = product == kOpI8 ? 1 : 2;
  LinArgs a = {};
  a.P = static_cast<const char*>(W);
  a.Q = static_cast<const char*>(X);
  a.ldp = mx4 ? K / 2 : mx8 ? K : es * ldw;
  a.ldq = es * ldx;
  a.p_group = mx4 || mx8 ? a.ldp * N : es * w_group;
  a.offsets = grouped ? &some_list : nullptr;
  a.M = n_entries;
  a.n_rows = n_entries;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(dgrad ? K : N);
  a.nc = static_cast<int>(dgrad ? N : K);
  RowsChoice c;
  switch (product) {
    case 0: c = choose_rows<kOpBF16, kLinForward>(a); break;
    case 1: c = choose_rows<kOpF16, kLinForward>(a); break;
    case 2: c = choose_rows<kOpI8, kLinForward>(a); break;
    case 3: c = choose_rows<kOpMx4, kLinForward>(a); break;
    case 4: c = choose_rows<kOpMx8, kLinForward>(a); break;
    case 5: c = choose_rows<kOpBF16, kLinDgrad>(a); break;
    default: c = choose_rows<kOpF16, kLinDgrad>(a); break;
  }
  MGQ_REQUIRE(c.nq || c.tile.rows, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  tile[0] = c.nq ? 16 * c.nq : c.tile.rows;
  tile[1] = c.nq ? lin_few_cols(c.nq) : c.tile.cols;
  tile[2] = c.nq ? 0 : c.tile.staged ? 2 : 1;
  return MGQ_OK;
}
