// Second launch of a routed layer for a few rows (experts_decode.h): down projection and
// the weighted sum over each row's experts, and the entry point of both.
//
// A workgroup computes 32 columns of the result for all rows. Its waves take the plan's items
// in turn (an expert with up to 16 of its rows) and add what an item gives each row into sums
// of their own in LDS; these are added in wave order. Where the columns alone would leave
// CUs without work, several workgroups share the items of a column tile and the last one of
// them to come adds their sums, in a fixed order. A single row needs no plan: its items are
// its entries (gemv_core.h).
//
// 128 experts of 2048 x 768: 68 us for 64 rows of MXFP8 (207 MB, 3.0 TB/s), 18 us for 16 rows
// of 4-bit codes (25 MB: the plan's read, the zeroed sums and the join are 5 us of it). Two waves
// a SIMD (173 to 254 registers) wait for 56 % of their cycles, vector instructions are 7 of the
// 68 us. One row 5.8 us in bf16 (25 MB), 3.4 in MXFP4.
#include "experts_decode.h"

namespace mgq {
namespace {

constexpr int kWaves = 4;

// Where the activation has two parts, both are rows of the MFMA: up to 4 rows in the call
// (NE = 2) row 4 j + i is part i of an item's row j, otherwise row 8 i + j is.
template <class F, int NE, int DEPTH>
__global__ void __launch_bounds__(64 * kWaves) decode_down_kernel(const DecodeArgs a) {
  constexpr int NP = kDecodeCols / 16;
  extern __shared__ float lds[];
  __shared__ __attribute__((aligned(16))) char params[F::dense ? 16 : kWaves * few_lds<F, NP>()];
  __shared__ int32_t done;
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x / a.parts, part = blockIdx.x - tile * a.parts;
  const int h0 = tile * kDecodeCols;
  float* sums = lds + wave * a.T * kDecodeCols;  // [T][32]
  DecodeItem* items = reinterpret_cast<DecodeItem*>(lds + kWaves * a.T * kDecodeCols);
  DecodeEntry* entries = reinterpret_cast<DecodeEntry*>(items + a.n);
  char* own_params = params + (F::dense ? 0 : wave * few_lds<F, NP>());
  for (int i = lane; i < a.T * kDecodeCols; i += 64) sums[i] = 0.0f;
  const int n_items = __builtin_amdgcn_readfirstlane(a.plan[0]);
  const uint64_t* from = reinterpret_cast<const uint64_t*>(a.plan + kDecodePlanHead / 4);
  for (int i = threadIdx.x; i < 2 * a.n; i += 64 * kWaves) reinterpret_cast<uint64_t*>(items)[i] = from[i];
  __syncthreads();

  const int whole = a.I / kFewStep, steps = (a.I + kFewStep - 1) / kFewStep;
  const int shift = F::affine ? a.down.shift : 5, groups = a.I >> shift;
  const int period = (kFewGroups << shift) / kFewStep;
  const int unit0 = part * kWaves + wave, stride = a.parts * kWaves;
  auto rows_of = [&](int u, FewRow(&row)[NP]) {
    const int expert = __builtin_amdgcn_readfirstlane(items[u].expert);
#pragma unroll
    for (int p = 0; p < NP; ++p)
      row[p] = few_row<F>(a.down, expert, h0 + 16 * p < a.H ? h0 + 16 * p : a.H - 1, a.I);
  };
  auto x_of = [&](int u) {
    const int first = __builtin_amdgcn_readfirstlane(items[u].first);
    const int count = __builtin_amdgcn_readfirstlane(items[u].count);
    const bool two = NE == 2 || a.act_parts == 2;
    const int own = NE == 2 ? r16 >> 2 : two ? r16 & 7 : r16;
    const int part = NE == 2 ? r16 & 1 : two ? r16 >> 3 : 0;
    const int64_t entry = entries[first + (own < count ? own : count - 1)].entry;
    return reinterpret_cast<const char*>(a.act + (entry * (two ? 2 : 1) + part) * a.I);
  };
  // an item's sums to its rows
  auto add = [&](int u, const lin_f32x4_t(&acc)[NP][1]) {
    const int first = __builtin_amdgcn_readfirstlane(items[u].first);
    const int count = __builtin_amdgcn_readfirstlane(items[u].count);
    constexpr int N = NE == 2 ? 1 : NE;
    float v[NP][N];
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int e = 0; e < N; ++e) v[p][e] = NE == 2 ? acc[p][0][0] + acc[p][0][1] : acc[p][0][e];
    if (NE == 4 && a.act_parts == 2) {  // (the upper half of the wave has the other parts)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const auto s = __builtin_amdgcn_permlane32_swap(f2u(v[p][e]), f2u(v[p][e]), false, false);
          v[p][e] = u2f(s[0]) + u2f(s[1]);
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int j = NE == 2 ? quad : 4 * quad + e;
      if (j < count) {  // (an item holds a row once: no two lanes add to one sum)
        const DecodeEntry t = entries[first + j];
        float* to = sums + t.entry / a.k * kDecodeCols + r16;
#pragma unroll
        for (int p = 0; p < NP; ++p) to[16 * p] += t.weight * v[p][e];
      }
    }
  };
  if (whole == 0) {
    for (int u = unit0; u < n_items; u += stride) {
      FewRow row[NP];
      rows_of(u, row);
      const char* const x[1] = {x_of(u)};
      lin_f32x4_t acc[NP][1];
      few_product<F, NP, 1, NE, 2>(row, a.down, x, a.I, 0, steps, own_params, acc);
      add(u, acc);
    }
  } else if (unit0 < n_items) {
    // The wave's items one after the other as one stream of steps, so that the next item's
    // operands are on their way while one ends.
    FewStep<F> f[DEPTH][NP];
    lin_u32x4_t xv[DEPTH][1][4];
    FewRow load_row[NP], row[NP];
    FewParams<F> par[NP];
    int lu = unit0, ls = 0;  // what is loaded next
    rows_of(lu, load_row);
    const char* lx = x_of(lu);
    auto load = [&](int d) __attribute__((always_inline)) {
      if (lu >= n_items) return;
#pragma unroll
      for (int p = 0; p < NP; ++p) few_load<F, true>(f[d][p], load_row[p], ls, a.I);
      few_load_x<F, true>(xv[d][0], lx, ls, a.I);
      if (++ls == whole) {
        ls = 0;
        lu += stride;
        if (lu < n_items) {
          rows_of(lu, load_row);
          lx = x_of(lu);
        }
      }
    };
    auto fetch = [&](const FewRow(&r)[NP], int g) __attribute__((always_inline)) {
      if constexpr (!F::dense) {
#pragma unroll
        for (int p = 0; p < NP; ++p) few_fetch<F>(par[p], r[p], g, groups);
      }
    };
    int u = unit0, s = 0, group = 0;
    rows_of(u, row);
    fetch(row, 0);
    lin_f32x4_t acc[NP][1];
    auto clear = [&]() {
#pragma unroll
      for (int p = 0; p < NP; ++p) acc[p][0] = lin_f32x4_t{0, 0, 0, 0};
    };
    clear();
    auto stage = [&](int at) __attribute__((always_inline)) {
      if constexpr (!F::dense) {
        if ((at & (period - 1)) == 0) {
          few_stage<F, NP>(par, a.down.type, own_params);
          group = at * kFewStep >> shift;
          if (at + period < steps) {
            fetch(row, (at + period) * kFewStep >> shift);
          } else if (u + stride < n_items) {
            FewRow next[NP];
            rows_of(u + stride, next);
            fetch(next, 0);
          }
        }
      }
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) load(d);
    const int total = (n_items - unit0 + stride - 1) / stride * whole;
    for (int at = 0; at < total; at += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        if (at + d >= total) break;
        load((d + DEPTH - 1) % DEPTH);
        stage(s);
        few_multiply<F, NP, 1, NE, true>(f[d], xv[d], s, a.I, shift, (s * kFewStep >> shift) - group,
                                         own_params, acc);
        if (++s < whole) continue;
        if (whole < steps) {
          FewStep<F> tail[NP];
          lin_u32x4_t tx[1][4];
#pragma unroll
          for (int p = 0; p < NP; ++p) few_load<F, false>(tail[p], row[p], whole, a.I);
          few_load_x<F, false>(tx[0], x_of(u), whole, a.I);
          stage(whole);
          few_multiply<F, NP, 1, NE, false>(tail, tx, whole, a.I, shift, (whole * kFewStep >> shift) - group,
                                            own_params, acc);
        }
        add(u, acc);
        clear();
        s = 0;
        u += stride;
        if (u < n_items) rows_of(u, row);
      }
    }
  }
  __syncthreads();
  const int outputs = a.T * kDecodeCols;
  auto wave_sum = [&](int i) {
    float sum = lds[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += lds[w * outputs + i];
    return sum;
  };
  auto store = [&](int i, float v) {
    const int col = h0 + i % kDecodeCols;
    if (col < a.H) a.out[static_cast<int64_t>(i / kDecodeCols) * a.H + col] = lin_round16(v, a.type);
  };
  if (a.parts == 1) {
    for (int i = threadIdx.x; i < outputs; i += 64 * kWaves) store(i, wave_sum(i));
    return;
  }
  // The workgroup that comes last adds the parts, in their order. They go past the XCDs'
  // L2s in stores and loads of their own, each waited for: a fence would write back and
  // invalidate the whole L2 for every workgroup (158 instead of 69 us for 64 rows of MXFP8).
  float* mine = a.sums + (static_cast<int64_t>(tile) * a.parts + part) * outputs;
  for (int i = threadIdx.x; i < outputs; i += 64 * kWaves)
    __hip_atomic_store(mine + i, wave_sum(i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  lds_handover();  // every wave's stores have arrived
  if (threadIdx.x == 0)
    done = __hip_atomic_fetch_add(a.counts + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (done != a.parts - 1) return;
  const float* all = a.sums + static_cast<int64_t>(tile) * a.parts * outputs;
  for (int i = threadIdx.x; i < outputs; i += 64 * kWaves) {
    float sum = 0.0f;
    for (int o = 0; o < a.parts; ++o)
      sum += __hip_atomic_load(all + o * outputs + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    store(i, sum);
  }
}

template <class F, int NE>
int launch(const DecodeArgs& a, hipStream_t s, const char* what) {
  decode_down_kernel<F, NE, 3><<<static_cast<unsigned>(a.tiles * a.parts), 64 * kWaves,
                                 kWaves * a.T * kDecodeCols * 4 + 16 * a.n, s>>>(a);
  return check_launch(what);
}

// A single row: a workgroup takes R 64 / L columns of the result, its waves the row's
// experts in turn (parts of the contraction where there are fewer experts than waves).
template <class F, int L, int R, int WAVES, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES) decode_down_single_kernel(const DecodeArgs a, const int parts) {
  constexpr int RI = 64 / L, ROWS = R * RI, N = gemv_sums<L, R>();
  __shared__ float sums[WAVES][ROWS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h0 = blockIdx.x * ROWS;
  auto first = [&](int r) { return h0 + r * RI < a.H - RI ? h0 + r * RI : a.H - RI; };
  const int chunks = gemv_chunks<F, L>(a.I);
  float acc[R], sum[N];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.0f;
  for (int u = wave; u < a.n * parts; u += WAVES) {
    const int i = u / parts, part = u - i * parts;
    const int expert = __builtin_amdgcn_readfirstlane(decode_expert(a, i));
    if (expert < 0) continue;
    const float weight = a.weights[i];
    float one[R];
#pragma unroll
    for (int r = 0; r < R; ++r) one[r] = 0.0f;
    gemv_add<F, L, R, DEPTH, 2>(one, a.down, expert, first,
                                reinterpret_cast<const char*>(a.act + static_cast<int64_t>(i) * 2 * a.I),
                                a.I, chunks * part / parts, chunks * (part + 1) / parts);
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = fmaf(weight, one[r], acc[r]);
  }
  gemv_reduce<L, R>(acc, sum);
#pragma unroll
  for (int q = 0; q < N; ++q)
    if ((lane & 15) == q) sums[wave][gemv_row<L>(q, lane >> 4)] = sum[q];
  __syncthreads();
  const int r = threadIdx.x;
  if (r < ROWS) {
    float v = sums[0][r];
#pragma unroll
    for (int o = 1; o < WAVES; ++o) v += sums[o][r];
    a.out[first(r / RI) + r % RI] = lin_round16(v, a.type);
  }
}

constexpr int kSingleWaves = 8;
constexpr int single_loads(int lanes) { return lanes == 64 ? 8 : 4; }

template <class F, int L>
int launch_single(const DecodeArgs& a, hipStream_t s, const char* what) {
  constexpr int R = single_loads(L), WAVES = kSingleWaves, DEPTH = F::dense ? 3 : 2;
  const int chunks = gemv_chunks<F, L>(a.I);
  int parts = WAVES / a.n;
  parts = parts < 1 ? 1 : parts > chunks ? chunks : parts;
  decode_down_single_kernel<F, L, R, WAVES, DEPTH>
      <<<static_cast<unsigned>(ceil_div(a.H, R * (64 / L))), 64 * WAVES, 0, s>>>(a, parts);
  return check_launch(what);
}

// Less than 2^32 threads (of several rows always: H < 2^29 are less than 2^24 tiles).
int check_grid(const DecodeArgs& a, int format, const char* what) {
  if (a.T > 1) return MGQ_OK;
  return decode_dispatch(format, a.type, a.down.type, [&](auto f) {
    const int lanes = gemv_lanes<decltype(f)>(a.I, a.H);
    const int64_t blocks = ceil_div(a.H, single_loads(lanes) * (64 / lanes));
    MGQ_REQUIRE(blocks < (int64_t(1) << 32) / (64 * kSingleWaves), MGQ_ERR_SHAPE,
                "%s: too many output tiles", what);
    return static_cast<int>(MGQ_OK);
  });
}

}  // namespace

int decode_down(const DecodeArgs& a, int format, hipStream_t s, const char* what) {
  return decode_dispatch(format, a.type, a.down.type, [&](auto f) {
    using F = decltype(f);
    if (a.T == 1) {
      const int lanes = gemv_lanes<F>(a.I, a.H);
      return lanes == 64   ? launch_single<F, 64>(a, s, what)
             : lanes == 32 ? launch_single<F, 32>(a, s, what)
                           : launch_single<F, 16>(a, s, what);
    }
    return a.T <= 4 ? launch<F, 2>(a, s, what) : launch<F, 4>(a, s, what);
  });
}

}  // namespace mgq

using namespace mgq;

extern "C" int64_t mgq_experts_decode_workspace_size(int64_t T, int64_t k, int64_t H, int64_t I) {
  if (T < 1 || k < 1 || H < 1 || I < 1) return 0;
  const int64_t n = T * k, parts = decode_parts(n, H);
  return decode_act_bytes(T, k, I) + decode_plan_bytes(n) + decode_count_bytes(H) +
         (parts > 1 ? parts * T * decode_tiles(H) * kDecodeCols * 4 : 0);
}

extern "C" int mgq_experts_decode(const void* X, int dtype, int64_t T, int64_t ldx, const void* index,
                                  int index_bits, const float* weights, int64_t k, int64_t n_experts,
                                  int64_t H, int64_t I, const mgq_weight* up, const mgq_weight* down,
                                  void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* what = "experts_decode";
  MGQ_REQUIRE(dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE, "%s: bfloat16 or float16 rows only", what);
  MGQ_REQUIRE(index_bits == 32 || index_bits == 64, MGQ_ERR_VALUE, "%s: 32- or 64-bit expert ids", what);
  MGQ_REQUIRE(T >= 0 && T <= kDecodeRows, MGQ_ERR_SHAPE, "%s: %lld rows (at most %d)", what,
              (long long)T, kDecodeRows);
  MGQ_REQUIRE(k >= 1 && k <= kDecodeTopK, MGQ_ERR_SHAPE, "%s: %lld experts a row (1 .. %d)", what,
              (long long)k, kDecodeTopK);
  MGQ_REQUIRE(n_experts >= 1 && n_experts <= (int64_t(1) << 20), MGQ_ERR_SHAPE,
              "%s: %lld experts (1 .. 2^20)", what, (long long)n_experts);
  MGQ_REQUIRE(H >= 1 && I >= 1 && H < (int64_t(1) << 29) && I < (int64_t(1) << 29), MGQ_ERR_SHAPE,
              "%s: bad layer sizes %lld, %lld", what, (long long)H, (long long)I);
  MGQ_REQUIRE(ldx >= H, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  auto weight = [&](const mgq_weight& m, int64_t n, int64_t cols, FewWeight* w) -> int {
    const int format = m.format;
    MGQ_REQUIRE(format >= kFewDense && format <= kFewAf8, MGQ_ERR_VALUE, "%s: no such weight format",
                what);
    MGQ_REQUIRE(dtype == kBF16 || (format != kFewMx4 && format != kFewMx8), MGQ_ERR_VALUE,
                "%s: MXFP weights take bfloat16 rows", what);
    MGQ_REQUIRE(m.data != nullptr, MGQ_ERR_VALUE, "%s: a weight has no elements", what);
    w->p = static_cast<const char*>(m.data);
    w->n = n;
    if (format == kFewDense) {
      MGQ_REQUIRE(m.ld >= cols && m.ld <= kFewRowBytes / 2, MGQ_ERR_SHAPE,
                  "%s: a weight's pitch is shorter than its row, or passes 2^28 bytes", what);
      w->ld = 2 * m.ld;
      w->group = 2 * m.expert;
      return MGQ_OK;
    }
    w->s = static_cast<const char*>(m.scales);
    w->b = static_cast<const char*>(m.biases);
    const int bits = format == kFewAf2 ? 2 : format == kFewMx4 || format == kFewAf4 ? 4 : 8;
    int64_t group = kMxGroup;
    if (format >= kFewAf2) {
      group = m.group;
      MGQ_REQUIRE(group == 32 || group == 64 || group == 128, MGQ_ERR_VALUE,
                  "%s: groups of 32, 64 or 128 values", what);
      MGQ_REQUIRE(m.param_dtype == kF32 || m.param_dtype == kBF16 || m.param_dtype == kF16,
                  MGQ_ERR_VALUE, "%s: scales and biases are float32, bfloat16 or float16", what);
      w->shift = group == 32 ? 5 : group == 64 ? 6 : 7;
      w->type = m.param_dtype;
    }
    MGQ_REQUIRE(cols % group == 0, MGQ_ERR_SHAPE, "%s: %lld columns are no multiple of the group size",
                what, (long long)cols);
    w->ld = cols / 8 * bits;
    MGQ_REQUIRE(w->ld <= kFewRowBytes, MGQ_ERR_SHAPE, "%s: a weight's rows pass 2^28 bytes", what);
    MGQ_REQUIRE(m.scales != nullptr && (format < kFewAf2 || m.biases != nullptr), MGQ_ERR_VALUE,
                "%s: a weight has no scales, or an affine one no biases", what);
    w->group = w->ld * n;
    return MGQ_OK;
  };
  MGQ_REQUIRE(up != nullptr && down != nullptr, MGQ_ERR_VALUE, "%s: a weight's description is missing",
              what);
  DecodeArgs a = {};
  if (int rc = weight(*up, 2 * I, H, &a.up)) return rc;
  if (int rc = weight(*down, H, I, &a.down)) return rc;
  const int64_t need = mgq_experts_decode_workspace_size(T, k, H, I);
  MGQ_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), MGQ_ERR_WORKSPACE,
              "%s: workspace %lld < %lld bytes", what, (long long)(workspace ? workspace_bytes : 0),
              (long long)need);
  if (T == 0) return MGQ_OK;
  a.x = static_cast<const char*>(X);
  a.ldx = 2 * ldx;
  a.index = index;
  a.index64 = index_bits == 64;
  a.weights = weights;
  a.act = static_cast<uint16_t*>(workspace);
  a.act_parts = decode_act_parts(T);
  a.plan = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + decode_act_bytes(T, k, I));
  a.counts = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(a.plan) + decode_plan_bytes(T * k));
  a.sums = reinterpret_cast<float*>(reinterpret_cast<char*>(a.counts) + decode_count_bytes(H));
  a.out = static_cast<uint16_t*>(out);
  a.T = static_cast<int>(T);
  a.k = static_cast<int>(k);
  a.n = static_cast<int>(T * k);
  a.E = static_cast<int>(n_experts);
  a.H = static_cast<int>(H);
  a.I = static_cast<int>(I);
  a.type = dtype;
  a.parts = decode_parts(T * k, H);
  a.tiles = decode_tiles(H);
  if (int rc = check_grid(a, down->format, what)) return rc;  // (before the first launch)
  hipStream_t s = as_stream(stream);
  if (int rc = decode_up(a, up->format, s, what)) return rc;
  return decode_down(a, down->format, s, what);
}
