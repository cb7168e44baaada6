// Second launch of a routed layer for a few rows (experts_decode.h): down projection and
// the weighted sum over each row's experts, and the entry point of both.
//
// A workgroup computes 16 columns of the result for all rows, so that no sum crosses
// workgroups. Its waves take the plan's items in turn (an expert with up to 16 of its
// rows; parts of the contraction where there are fewer items than waves) and add what an
// item gives each row into sums of their own in LDS; these are added in wave order. A
// single row needs no plan: its items are its entries (gemv_core.h).
#include "experts_decode.h"

namespace mgq {
namespace {

template <class F, int NE, int WAVES, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES) decode_down_kernel(const DecodeArgs a) {
  extern __shared__ float lds[];
  __shared__ __attribute__((aligned(16))) char params[F::dense ? 16 : WAVES * few_lds<F, 1>()];
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float* sums = lds + wave * a.T * 16;  // [T][16]
  DecodeItem* items = reinterpret_cast<DecodeItem*>(lds + WAVES * a.T * 16);
  DecodeEntry* entries = reinterpret_cast<DecodeEntry*>(items + a.n);
  for (int i = lane; i < a.T * 16; i += 64) sums[i] = 0.0f;
  const int n_items = __builtin_amdgcn_readfirstlane(a.plan[0]);
  const uint64_t* from = reinterpret_cast<const uint64_t*>(a.plan + kDecodePlanHead / 4);
  for (int i = threadIdx.x; i < 2 * a.n; i += 64 * WAVES) reinterpret_cast<uint64_t*>(items)[i] = from[i];
  __syncthreads();
  const int h0 = blockIdx.x * 16;
  const int steps = (a.I + kFewStep - 1) / kFewStep;
  for (int i = wave; i < n_items; i += WAVES) {
    const DecodeItem it = items[i];
    const int expert = __builtin_amdgcn_readfirstlane(it.expert);
    const int first = __builtin_amdgcn_readfirstlane(it.first);
    const int count = __builtin_amdgcn_readfirstlane(it.count);
    const FewRow row[1] = {few_row<F>(a.down, expert, h0, a.I)};
    const int own = NE == 1 ? r16 >> 2 : r16;
    const int entry = entries[first + (own < count ? own : count - 1)].entry;
    const char* const x[1] = {a.act + static_cast<int64_t>(entry) * a.I * 2};
    lin_f32x4_t acc[1][1];
    few_product<F, 1, 1, NE, DEPTH>(row, a.down, x, a.I, 0, steps, params + wave * few_lds<F, 1>(), acc);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int j = NE == 1 ? quad : 4 * quad + e;
      if (j < count) {  // (an item holds a row once: no two lanes add to one sum)
        const DecodeEntry t = entries[first + j];
        sums[t.entry / a.k * 16 + r16] += t.weight * acc[0][0][e];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.T * 16; i += 64 * WAVES) {
    const int col = blockIdx.x * 16 + (i & 15);
    if (col >= a.H) continue;
    float sum = lds[i];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += lds[w * a.T * 16 + i];
    a.out[static_cast<int64_t>(i >> 4) * a.H + col] = lin_round16(sum, a.type);
  }
}

template <class F, int NE, int WAVES, int DEPTH>
int launch(const DecodeArgs& a, hipStream_t s, const char* what) {
  decode_down_kernel<F, NE, WAVES, DEPTH>
      <<<static_cast<unsigned>(ceil_div(a.H, 16)), 64 * WAVES, WAVES * a.T * 64 + 16 * a.n, s>>>(a);
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
    gemv_add<F, L, R, DEPTH>(one, a.down, expert, first, a.act + static_cast<int64_t>(i) * a.I * 2, a.I,
                             chunks * part / parts, chunks * (part + 1) / parts);
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

template <class F, int L>
int launch_single(const DecodeArgs& a, hipStream_t s, const char* what) {
  constexpr int R = L == 64 ? 8 : 4, WAVES = 8, DEPTH = F::dense ? 3 : 2;
  const int chunks = gemv_chunks<F, L>(a.I);
  int parts = WAVES / a.n;
  parts = parts < 1 ? 1 : parts > chunks ? chunks : parts;
  decode_down_single_kernel<F, L, R, WAVES, DEPTH>
      <<<static_cast<unsigned>(ceil_div(a.H, R * (64 / L))), 64 * WAVES, 0, s>>>(a, parts);
  return check_launch(what);
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
    if (a.T <= 4) return launch<F, 1, 8, 3>(a, s, what);
    return launch<F, 4, 8, 3>(a, s, what);
  });
}

}  // namespace mgq

using namespace mgq;

extern "C" int64_t mgq_experts_decode_workspace_size(int64_t T, int64_t k, int64_t I) {
  if (T < 1 || k < 1 || I < 1) return 0;
  return decode_act_bytes(T * k, I) + decode_plan_bytes(T * k);
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
    w->p = static_cast<const char*>(m.data);
    w->n = n;
    if (format == kFewDense) {
      MGQ_REQUIRE(m.ld >= cols && m.ld < (int64_t(1) << 29), MGQ_ERR_SHAPE,
                  "%s: a weight's pitch is shorter than its row, or 2^29 elements", what);
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
    w->group = w->ld * n;
    return MGQ_OK;
  };
  DecodeArgs a = {};
  if (int rc = weight(*up, 2 * I, H, &a.up)) return rc;
  if (int rc = weight(*down, H, I, &a.down)) return rc;
  const int64_t need = mgq_experts_decode_workspace_size(T, k, I);
  MGQ_REQUIRE(workspace_bytes >= need, MGQ_ERR_WORKSPACE, "%s: workspace %lld < %lld bytes", what,
              (long long)workspace_bytes, (long long)need);
  if (T == 0) return MGQ_OK;
  a.x = static_cast<const char*>(X);
  a.ldx = 2 * ldx;
  a.index = index;
  a.index64 = index_bits == 64;
  a.weights = weights;
  a.act = static_cast<char*>(workspace);
  a.plan = reinterpret_cast<int32_t*>(a.act + decode_act_bytes(T * k, I));
  a.out = static_cast<uint16_t*>(out);
  a.T = static_cast<int>(T);
  a.k = static_cast<int>(k);
  a.n = static_cast<int>(T * k);
  a.E = static_cast<int>(n_experts);
  a.H = static_cast<int>(H);
  a.I = static_cast<int>(I);
  a.type = dtype;
  hipStream_t s = as_stream(stream);
  if (int rc = decode_up(a, up->format, s, what)) return rc;
  return decode_down(a, down->format, s, what);
}
