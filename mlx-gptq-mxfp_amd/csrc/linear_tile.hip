// Large tiles of the matrix products: the choice among the instances of the tile kernel
// (linear_tile_kernel.h) for dense, MX and int8 operands, the weight gradient's work list and
// the sum of its partial tiles. Affine weights are in affine_tile.hip.
#include "linear_tile_kernel.h"

namespace mgq {
namespace {

// A cap that no group is longer than.
constexpr int kLinNoCap = 0x7fffffc0;

// ---------------------------------------------------------------------------
// wgrad's units: a group's entries, cut into chunks of at most `cap`, longest
// first so that the last tiles to start are the shortest. One workgroup plans. Each
// of its 16 waves prices one cap, cap_min 2^(k / 2): a CU takes about 1.5 us for 64
// entries of a tile and 5 us beside them, a cut tile's partial results cost the chip
// 0.11 us of memory traffic; the tiles of one round end with the longest, those of
// several about half the longest after the average load. Then a wave per group
// at a time: each place in the order is a sum over all groups. 8 groups take 4.4 us and
// 128 groups 11 us, which is latency. The prices are those of the 256 x 256 tile, also for
// rows off 16-byte boundaries, whose 128 x 256 tile takes 1.75 us for 64 entries.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) lin_plan_kernel(const LinArgs a, const LinPlanArgs pl) {
  __shared__ int32_t size[kLinPlanGroups], parts[kLinPlanGroups], chunk[kLinPlanGroups];
  __shared__ float price[16];
  __shared__ bool fits[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int g = threadIdx.x; g < a.G; g += 1024) {
    int64_t b = 0, e = a.M;
    if (a.offsets) lin_segment(a, g, &b, &e);
    size[g] = e > b ? static_cast<int>(e - b) : 0;
  }
  __syncthreads();
  auto cap_of = [&](int k) {  // a multiple of 64
    const int64_t c = (static_cast<int64_t>(pl.cap) << (k >> 1)) * (k & 1 ? 181 : 128) / 128;
    return static_cast<int>(c < kLinNoCap ? c & ~int64_t(63) : kLinNoCap);
  };
  {
    const int cap = cap_of(wave), tiles = pl.npt * pl.nqt;
    float load = 0, longest = 0;
    uint32_t units = 0, cut = 0, splits = 0;
    for (int o0 = 0; o0 < a.G; o0 += 64) {
      const int n = o0 + lane < a.G ? size[o0 + lane] : 0;
      const int k = n > cap ? (n - 1) / cap + 1 : 1;
      const float us = 5.0f + 1.5f / 64 * ((n + k - 1) / k);
      if (o0 + lane < a.G) {
        load += k * us;
        longest = fmaxf(longest, us);
        units += k;
        cut += k > 1 ? k : 0;
        splits += k > 1;
      }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      load += __shfl_xor(load, d);
      longest = fmaxf(longest, __shfl_xor(longest, d));
      units += __shfl_xor(units, d);
      cut += __shfl_xor(cut, d);
      splits += __shfl_xor(splits, d);
    }
    const float items = static_cast<float>(units) * tiles;
    const float us = (items <= 256 ? longest : load * tiles / 256 + 0.5f * longest) +
                     0.11f * cut * tiles;
    if (lane == 0) {
      price[wave] = us;
      fits[wave] = units <= static_cast<uint32_t>(pl.max_units) &&
                   cut <= static_cast<uint32_t>(pl.max_slots) &&
                   splits <= static_cast<uint32_t>(pl.max_splits);
    }
  }
  __syncthreads();
  int pick = 15;  // the longest cap among the cheapest
  for (int k = 14; k >= 0; --k) pick = price[k] < 0.97f * price[pick] ? k : pick;
  // (the workspace has room for the cuts of any list; groups whose offsets decrease may
  // overlap and add up to more: they stay whole)
  const int cap = fits[pick] ? cap_of(pick) : kLinNoCap;
  for (int g = threadIdx.x; g < a.G; g += 1024) {
    const int n = size[g];
    const int k = n > cap ? (n - 1) / cap + 1 : 1;
    parts[g] = k;
    chunk[g] = ((n + k - 1) / k + 63) & ~63;  // whole stages
  }
  __syncthreads();
  for (int g = wave; g < a.G; g += 16) {
    const int n = size[g], k = parts[g], len = chunk[g];
    // units before this group's, and its first slot, 16 bits each (there are at
    // most 4096 groups and 1025 cuts)
    uint32_t sums = 0, splits = 0, units = 0, all_splits = 0;
    for (int o0 = 0; o0 < a.G; o0 += 64) {
      const int o = o0 + lane;
      const int lo = o < a.G ? chunk[o] : -1;
      const uint32_t un = o < a.G ? parts[o] : 0;
      const bool before = o < g;
      const uint32_t own = (lo > len || (lo == len && before) ? un << 16 : 0) +
                           (before && un > 1 ? un : 0);
      sums += __builtin_amdgcn_readlane(lin_wave_scan(own), 63);
      splits += __popcll(__ballot(before && un > 1));
      if (g == 0) {
        units += __builtin_amdgcn_readlane(lin_wave_scan(un), 63);
        all_splits += __popcll(__ballot(un > 1));
      }
    }
    const uint32_t first = sums >> 16, slots = sums & 0xffffu;
    int64_t b = 0, e = a.M;
    if (a.offsets) lin_segment(a, g, &b, &e);
    for (int i = lane; i < k; i += 64) {
      const int64_t t0 = static_cast<int64_t>(i) * len, t1 = t0 + len;
      LinUnit u;
      u.g = g;
      u.t0 = static_cast<int32_t>(b + (t0 < n ? t0 : n));
      u.t1 = static_cast<int32_t>(b + (t1 < n ? t1 : n));
      u.slot = k > 1 ? static_cast<int32_t>(slots) + i : -1;
      pl.units[first + i] = u;
    }
    if (lane == 0) {
      if (k > 1) {
        pl.splits[splits].g = g;
        pl.splits[splits].slot0 = static_cast<int32_t>(slots);
        pl.splits[splits].n = k;
      }
      if (g == 0) {
        pl.counts[0] = static_cast<int>(units);
        pl.counts[1] = static_cast<int>(all_splits);
      }
    }
  }
}

// Partial tiles summed in chunk order: grid (tiles * bq / 16, splits), 256
// threads, 16 rows of a tile each.
__global__ void __launch_bounds__(256) lin_reduce_kernel(const LinArgs a, const LinPlanArgs pl) {
  if (static_cast<int>(blockIdx.y) >= pl.counts[1]) return;
  const LinSplit sp = pl.splits[blockIdx.y];
  const int tiles = pl.npt * pl.nqt, subs = pl.bq / 16;
  const int tile = blockIdx.x / subs, sub = blockIdx.x % subs;
  const int q0 = tile % pl.nqt * pl.bq + sub * 16, p0 = tile / pl.nqt * 256;
  const int p = p0 + 4 * (threadIdx.x & 63);
  if (p >= a.np) return;
  const int osize = a.out_type == kF32 ? 4 : 2;
  const int64_t tile_size = static_cast<int64_t>(pl.bq) * 256;
  for (int r = threadIdx.x >> 6; r < 16; r += 4) {
    const int q = q0 + r;
    if (q >= a.nq) return;
    float v[4] = {0, 0, 0, 0};
    for (int i = 0; i < sp.n; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(
          pl.partials + (static_cast<int64_t>(sp.slot0 + i) * tiles + tile) * tile_size +
          (sub * 16 + r) * 256 + (p - p0));
      v[0] += f.x;
      v[1] += f.y;
      v[2] += f.z;
      v[3] += f.w;
    }
    lin_store4(a, a.out + (sp.g * a.o_group + q * a.ldo) * osize, p, v);
  }
}

template <int OP>
int launch_wgrad(const LinArgs& a, const LinPlanArgs& pl, bool staged, int64_t grid, hipStream_t s,
                 const char* what) {
  if (a.row_index)
    return staged ? launch<OP, kLinWgradGather, 2, 2, true>(a, pl, grid, s, what)
                  : launch<OP, kLinWgradGather, 4, 2, false>(a, pl, grid, s, what);
  return staged ? launch<OP, kLinWgrad, 2, 2, true>(a, pl, grid, s, what)
                : launch<OP, kLinWgrad, 4, 2, false>(a, pl, grid, s, what);
}

inline bool aligned16(const void* p, int64_t pitch) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (pitch & 15) == 0;
}

LinPlanSizes plan_sizes(int64_t M, int64_t G, int64_t N, int64_t K, int bq) {
  LinPlanSizes z;
  z.tiles = ceil_div(N, bq) * ceil_div(K, 256);
  const int64_t cap = M * z.tiles / 1024;  // at most 2048 partial tiles
  z.cap = cap < 256 ? 256 : cap < kLinNoCap ? (cap + 63) & ~int64_t(63) : kLinNoCap;
  const int64_t over = M / z.cap + 1;  // whole chunks, and groups longer than cap
  z.max_splits = M > z.cap ? (over < G ? over : G) : 0;
  z.max_slots = z.max_splits ? over + z.max_splits : 0;
  z.max_units = G + (z.max_splits ? over : 0);
  z.units_off = 256;
  z.splits_off = z.units_off + ceil_div(z.max_units * static_cast<int64_t>(sizeof(LinUnit)), 256) * 256;
  z.partials_off =
      z.splits_off + ceil_div(z.max_splits * static_cast<int64_t>(sizeof(LinSplit)), 256) * 256;
  z.bytes = z.partials_off + z.max_slots * z.tiles * bq * 256 * 4;
  return z;
}

}  // namespace

bool lin_tile_direct(const LinArgs& a, int op, int kind) {
  const int es = op == kOpI8 ? 1 : 2;
  if (!aligned16(a.Q, a.ldq) || !aligned16(a.P, a.ldp) || (a.p_group & 15)) return false;
  if (kind == kLinForward) return a.nc * es % 16 == 0;
  return (kind == kLinDgrad ? a.nc : a.nq) % 8 == 0 && a.np % 8 == 0;
}

int lin_tile_rows(const LinArgs& a, int op, int kind, LinTileShape t, hipStream_t s,
                  const char* what) {
  if (kind == kLinDgrad)
    return op == kOpF16 ? pick_rows<kOpF16, kLinDgrad>(a, t, s, what)
                        : pick_rows<kOpBF16, kLinDgrad>(a, t, s, what);
  switch (op) {
    case kOpBF16: return pick_rows<kOpBF16, kLinForward>(a, t, s, what);
    case kOpF16: return pick_rows<kOpF16, kLinForward>(a, t, s, what);
    case kOpI8: return pick_rows<kOpI8, kLinForward>(a, t, s, what);
    case kOpMx4: return pick_rows<kOpMx4, kLinForward>(a, t, s, what);
    case kOpMx8: return pick_rows<kOpMx8, kLinForward>(a, t, s, what);
    default: break;
  }
  set_error("%s: no such operands", what);  // (affine ones have lin_tile_affine)
  return MGQ_ERR_VALUE;
}

int64_t lin_tile_wgrad_bytes(int64_t M, int64_t G, int64_t N, int64_t K) {
  const int64_t a = plan_sizes(M, G, N, K, 128).bytes, b = plan_sizes(M, G, N, K, 256).bytes;
  return a > b ? a : b;
}

int lin_tile_wgrad(const LinArgs& a, int op, void* workspace, hipStream_t s, const char* what) {
  const bool staged = !lin_tile_direct(a, op, kLinWgrad);
  const int bq = staged ? 128 : 256;
  const LinPlanSizes z = plan_sizes(a.M, a.G, a.nq, a.np, bq);
  char* ws = static_cast<char*>(workspace);
  LinPlanArgs pl = {};
  pl.counts = reinterpret_cast<int32_t*>(ws);
  pl.units = reinterpret_cast<LinUnit*>(ws + z.units_off);
  pl.splits = reinterpret_cast<LinSplit*>(ws + z.splits_off);
  pl.partials = reinterpret_cast<float*>(ws + z.partials_off);
  pl.npt = static_cast<int>(ceil_div(a.np, 256));
  pl.nqt = static_cast<int>(ceil_div(a.nq, bq));
  pl.bq = bq;
  pl.cap = static_cast<int>(z.cap);
  pl.max_units = static_cast<int>(z.max_units);
  pl.max_splits = static_cast<int>(z.max_splits);
  pl.max_slots = static_cast<int>(z.max_slots);
  pl.deal = a.G >= 64;
  lin_plan_kernel<<<1, 1024, 0, s>>>(a, pl);
  if (int rc = check_launch(what)) return rc;
  const int64_t grid = (pl.deal ? ceil_div(z.max_units, 8) * 8 : z.max_units) * z.tiles;
  const int rc = op == kOpF16 ? launch_wgrad<kOpF16>(a, pl, staged, grid, s, what)
                              : launch_wgrad<kOpBF16>(a, pl, staged, grid, s, what);
  if (rc || z.max_splits == 0) return rc;
  const dim3 rg(static_cast<unsigned>(z.tiles * (bq / 16)), static_cast<unsigned>(z.max_splits));
  lin_reduce_kernel<<<rg, 256, 0, s>>>(a, pl);
  return check_launch(what);
}

}  // namespace mgq
