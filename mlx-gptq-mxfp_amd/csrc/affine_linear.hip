// Products with affine weights, y[t, n] = sum_k x[r(t), k] (q[g, n, k] s + b) with a scale
// s and a bias b for each group of 32, 64 or 128 values of a weight row and 2-, 4- or
// 8-bit codes q, packed low bits first. The list of entries t and its groups g are those of
// linear_common.h. Here are the entry point and the choice of kernel: affine_few.h for few
// rows, the tile kernel of the other products (affine_tile.hip) for many.
#include <math.h>

#include "affine_few_choice.h"
#include "linear_few.h"

namespace mgq {
namespace {

int run_tile(LinArgs a, const FewWeight& w, int bits, LinTileShape t, hipStream_t s, const char* what) {
  a.P = w.p;
  a.Ps = reinterpret_cast<const uint8_t*>(w.s);
  a.Pb = reinterpret_cast<const uint8_t*>(w.b);
  a.ldp = w.ld;
  a.p_group = w.group;
  a.p_shift = w.shift;
  a.p_type = w.type;
  const int op = (a.out_type == kF16 ? kOpAf2H : kOpAf2) + (bits == 8 ? 2 : bits == 4 ? 1 : 0);
  return lin_tile_affine(a, op, t, s, what);
}
int run_few(const LinArgs& a, const FewWeight& w, int bits, int choice, hipStream_t s, const char* what) {
  if (bits == 2) return affine_few_bits2(a, w, choice, s, what);
  if (bits == 4) return affine_few_bits4(a, w, choice, s, what);
  return affine_few_bits8(a, w, choice, s, what);
}

// The kernel whose time by the model below is least, of those whose grid holds the
// product. Times are of 4-bit codes with a scale for 64 values (one MI355X, called again and
// again with weights that had left the caches) and stand for the other codes too. With them
// 14336 x 4096 in 2, 4 and 8 bits takes 14.6, 15.4 and 19.8 us for 16 entries, 27.8, 27.7 and
// 32.7 for 64, 55.5, 54.8 and 55.2 for 128, 102, 99 and 99 for 512.
//   few rows: the steps of 128 values that a wave takes, one after the other, at the time
//     of a step for a wave alone on its SIMD or for the waves that share it (a form's
//     numbers in affine_few_choice.h), three more where workgroups follow one another;
//   single entries: chunks of 64 pieces of eight rows, 1.65 us each;
//   tiles: the stages of 64 values, rounds of the 256 CUs; up to 1.45 times as much when
//     every CU has one.
// Groups of unknown lengths are taken as in the other products (linear.hip). 14336 x 4096, 4
// bits: 1 entry 11 us (0), 4 entries 12.7 (1), 16 entries 15.6 (4; the largest tile 114), 64
// entries 28.8 (10; the smallest tile 58.7), 512 entries 103 (128 x 256; form 10: 210).
struct Choice {
  int few;
  LinTileShape tile;
};
Choice choose(const LinArgs& a, const FewWeight& w, int bits) {
  const double M = static_cast<double>(a.M), active = a.offsets ? (a.G < a.M ? a.G : M) : 1;
  const double steps = ceil_div(a.nc, kFewStep);
  auto row_tiles = [&](int rows) {
    return a.offsets ? fmax(1.0, M / rows + 0.575 * active) : ceil(M / rows);
  };
  Choice c = {};
  double best = 1e300;
  auto offer = [&](double us, int few, LinTileShape tile) {
    if (us < best) {
      best = us;
      c = Choice{few, tile};
    }
  };
  if (a.M * ceil_div(a.np, 32) < kLinFewGrid) {
    const double chunks = ceil_div(a.nc, bits == 8 ? 1024 : 2048);
    offer(5 + chunks * 1.65 * fmax(1.0, M * ceil_div(a.np, 8) / 1024.0), 0, LinTileShape{});
  }
#define MGQ_OFFER(n, NP, NQ, NE, WAVES, KS, depth, alone, shared)                      \
  {                                                                                    \
    constexpr int rows = NE == 1 ? 4 : 16 * NQ, cols = 16 * NP * (WAVES / KS);          \
    if (lin_row_tiles(a, rows) * ceil_div(a.np, cols) < kLinFewGrid * 4 / WAVES) {       \
      const double on_simd = row_tiles(rows) * ceil_div(a.np, cols) * WAVES / 1024;      \
      const double more = on_simd > 1 ? 3 * (1 - 1 / on_simd) : 0;                       \
      offer(5 + (ceil(steps / KS) + more) *                                              \
                    fmax(alone, shared * (on_simd + ceil(on_simd)) / 2),                 \
            n, LinTileShape{});                                                         \
    }                                                                                  \
  }
  MGQ_AFFINE_SHAPES(MGQ_OFFER)
#undef MGQ_OFFER
  // (a piece of 16 bytes of 2-bit codes holds 64 values: the rows have to)
  if (bits != 2 || a.nc % 64 == 0) {
    LinArgs t = a;
    t.P = w.p;
    t.ldp = w.ld;
    t.p_group = w.group;
    const bool staged = !lin_tile_direct(t, kOpAf4, kLinForward);
    struct {
      int rows, cols;
      double stage, full;
    } const tiles[] = {{64, 128, 0.64, 1.05}, {64, 256, 1.05, 1.0}, {128, 256, 1.22, 1.29},
                       {256, 256, 1.5, 1.45}};
    for (const auto& v : tiles) {
      if ((staged && v.rows == 256) || lin_tile_grid(a, v.rows, v.cols) >= kLinTileGrid) continue;
      const double rounds = row_tiles(v.rows) * ceil_div(a.np, v.cols) / 256;
      const double full = rounds > 1 ? v.full : 1.0;
      offer(5 + (rounds < 1 ? 1 : rounds + 0.617 * (ceil(rounds) - rounds)) *
                    (ceil_div(a.nc, 64) * v.stage * full * (staged ? 1.3 : 1.0) + 3),
            0, LinTileShape{v.rows, v.cols, staged});
    }
  }
  return c;
}

int run(const LinArgs& a, const FewWeight& w, int bits, hipStream_t s, const char* what) {
  const Choice c = choose(a, w, bits);
  if (c.tile.rows) return run_tile(a, w, bits, c.tile, s, what);
  return run_few(a, w, bits, c.few, s, what);
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
  MGQ_REQUIRE(K > 0 && K % group_size == 0, MGQ_ERR_SHAPE,
              "%s: K = %lld is no multiple of the group size", what, (long long)K);
  MGQ_REQUIRE(K / 8 * bits <= kFewRowBytes, MGQ_ERR_SHAPE, "%s: rows of K = %lld codes pass 2^28 bytes",
              what, (long long)K);
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
  return run(a, w, bits, as_stream(stream), what);
}

extern "C" int mgq_affine_choice(const void* X, int64_t ldx, int64_t n_entries, const uint32_t* words,
                                 int bits, int64_t n_groups, int64_t N, int64_t K, int grouped,
                                 int32_t* kernel) {
  clear_error();
  const char* what = "affine_choice";
  MGQ_REQUIRE(bits == 2 || bits == 4 || bits == 8, MGQ_ERR_VALUE, "%s: bits must be 2, 4 or 8", what);
  const int32_t some_list = 0;  // stands for offsets: the choice does not read them
  if (int rc = lin_check_list(what, grouped ? &some_list : nullptr, nullptr, n_groups, n_entries, n_entries))
    return rc;
  if (int rc = lin_check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(K > 0 && K % 32 == 0, MGQ_ERR_SHAPE, "%s: K = %lld is no multiple of 32", what, (long long)K);
  LinArgs a = {};
  a.Q = static_cast<const char*>(X);
  a.ldq = 2 * ldx;
  a.offsets = grouped ? &some_list : nullptr;
  a.M = n_entries;
  a.n_rows = n_entries;
  a.G = static_cast<int>(n_groups);
  a.np = static_cast<int>(N);
  a.nc = static_cast<int>(K);
  FewWeight w = {};
  w.p = reinterpret_cast<const char*>(words);
  w.ld = K / 8 * bits;
  w.group = w.ld * N;
  const Choice c = choose(a, w, bits);
  kernel[0] = c.tile.rows ? (c.tile.staged ? 3 : 2) : c.few ? 1 : 0;
  kernel[1] = c.tile.rows ? c.tile.rows : c.few;
  kernel[2] = c.tile.cols;
  return MGQ_OK;
}
