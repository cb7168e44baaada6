// First launch of a routed layer for a few rows (experts_decode.h): gate and up
// projection of every entry and their activation, and the plan for the second launch.
//
// A workgroup takes 16 gate rows and the 16 up rows beside them of one expert, with all
// entries of that expert: its weight is read once (again for every further 16 entries).
// The expert is that of list entry `slot`, whose workgroups end at once if an earlier
// entry has the same one, or, where there are more entries than experts, expert `slot`.
// The list is short enough for every wave to look through all of it.
#include "experts_decode.h"

namespace mgq {
namespace {

// One workgroup of 256: the entries in the experts' order. Thread e counts expert e's
// rows by walking the list, the counts are summed up over the experts, and a second walk
// writes. A row that names an expert twice is one entry with the sum of its weights.
__device__ void decode_plan(const DecodeArgs& a, int16_t* ids, uint32_t* carry) {
  typedef int16_t ids8_t __attribute__((ext_vector_type(8)));
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  DecodeItem* items = reinterpret_cast<DecodeItem*>(a.plan + kDecodePlanHead / 4);
  DecodeEntry* entries = reinterpret_cast<DecodeEntry*>(items + a.n);
  const uint32_t inv_k = 65536u / a.k + 1;  // i / k = i inv_k >> 16 (i < 1024, k <= 16)
  // f(entry, row) for the entries of this round's expert `tid`
  auto walk = [&](auto&& f) {
    for (int i = 0; i < a.n; i += 8) {
      const ids8_t v = *reinterpret_cast<const ids8_t*>(ids + i);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v[j] == tid) f(i + j, static_cast<int>((i + j) * inv_k >> 16));
    }
  };
  uint32_t base = 0;  // items << 16 | entries of the experts before this round's
  for (int e0 = 0; e0 < a.E; e0 += 256) {
    __syncthreads();
    // (relative to the round, so that 16 bits hold any number of experts)
    for (int i = tid; i < ((a.n + 7) & ~7); i += 256) {
      const int e = i < a.n ? decode_expert(a, i) - e0 : -1;
      ids[i] = static_cast<int16_t>(e >= 0 && e < 256 ? e : -1);
    }
    __syncthreads();
    uint32_t count = 0;
    int last = -1;
    walk([&](int, int row) {
      count += row != last;
      last = row;
    });
    const uint32_t own = (count + kDecodeItem - 1) / kDecodeItem << 16 | count;
    const uint32_t incl = lin_wave_scan(own);
    if (lane == 63) carry[wave] = incl;
    __syncthreads();
    uint32_t before = base;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += carry[w];
      base += carry[w];
    }
    before += incl - own;
    int item = before >> 16, at = before & 0xffff;
    for (uint32_t c = 0; c < count; c += kDecodeItem)
      items[item++] = DecodeItem{e0 + tid, static_cast<uint16_t>(at + c),
                                 static_cast<uint16_t>(count - c < kDecodeItem ? count - c : kDecodeItem)};
    last = -1;
    --at;
    walk([&](int i, int row) {
      const float w = a.weights[i];
      if (row != last) {
        last = row;
        entries[++at] = DecodeEntry{i, w};
      } else {
        entries[at].weight += w;
      }
    });
  }
  if (tid == 0) a.plan[0] = static_cast<int32_t>(base >> 16);
  for (int i = tid; i < a.tiles; i += 256) a.counts[i] = 0;
}

constexpr int kWaves = 4;

__device__ __forceinline__ float decode_act(float gate, float up) {
  return gate / (1.0f + expf(-gate)) * up;
}

// KS waves share the contraction; the others take 16 gate rows each.
template <class F, int NE, int KS, int DEPTH>
__global__ void __launch_bounds__(64 * kWaves) decode_up_kernel(const DecodeArgs a) {
  constexpr int BM = NE == 1 ? 4 : 16, BP = 16 * (kWaves / KS);
  __shared__ __attribute__((aligned(16))) int16_t list[kDecodeEntries];
  __shared__ uint32_t carry[kWaves];
  __shared__ lin_f32x4_t part[KS > 1 ? kWaves * 2 * 64 : 1];
  __shared__ __attribute__((aligned(16))) char params[F::dense ? 16 : kWaves * few_lds<F, 2>()];
  if (blockIdx.x == 0) {
    decode_plan(a, list, carry);
    return;
  }
  const int bid = blockIdx.x - 1;
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.I + BP - 1) / BP, kw = wave % KS;
  const int slot = bid / tiles, p0 = (bid - slot * tiles) * BP + wave / KS * 16, p = p0 + r16;
  const bool by_expert = a.n > a.E;
  const int expert = by_expert ? slot : __builtin_amdgcn_readfirstlane(decode_expert(a, slot));
  if (expert < 0) return;
  int count = 0;
  for (int c0 = 0; c0 < a.n; c0 += 512) {
    int ids[8];  // (loaded together: the list is the first thing that is waited for)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int i = c0 + 64 * c + lane;
      ids[c] = i < a.n ? decode_expert(a, i) : -1;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint64_t mask = __ballot(ids[c] == expert);
      const int i0 = c0 + 64 * c;
      if (!by_expert && count == 0 && mask && i0 + __builtin_ctzll(mask) < slot) return;
      if (wave == 0 && ids[c] == expert)
        list[count + __popcll(mask & ((uint64_t(1) << lane) - 1))] = static_cast<int16_t>(i0 + lane);
      count += __popcll(mask);
    }
  }
  if (count == 0) return;
  __syncthreads();

  FewRow row[2];
  // (a gate row past the last one is an up row, whose result is not stored)
  const int pc = p0 < a.I ? p0 : a.I - 1;
  row[0] = few_row<F>(a.up, expert, pc, a.H);
  row[1] = few_row<F>(a.up, expert, a.I + pc, a.H);
  const int steps = (a.H + kFewStep - 1) / kFewStep;
  for (int base = 0; base < count; base += BM) {
    const int j = base + (NE == 1 ? r16 >> 2 : r16);
    const int entry = list[j < count ? j : count - 1];
    const char* const x[1] = {a.x + entry / a.k * a.ldx};
    lin_f32x4_t acc[2][1];
    few_product<F, 2, 1, NE, DEPTH>(row, a.up, x, a.H, steps * kw / KS, steps * (kw + 1) / KS,
                                    params + wave * few_lds<F, 2>(), acc);
    lin_f32x4_t gate = acc[0][0], up = acc[1][0];
    if constexpr (KS > 1) {
      part[(2 * wave) * 64 + lane] = gate;
      part[(2 * wave + 1) * 64 + lane] = up;
      __syncthreads();
      if (kw == 0) {
#pragma unroll
        for (int w = 1; w < KS; ++w) {
          const lin_f32x4_t g = part[2 * (wave + w) * 64 + lane], u = part[(2 * (wave + w) + 1) * 64 + lane];
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            gate[e] += g[e];
            up[e] += u[e];
          }
        }
      }
    }
    if (kw == 0) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int i = base + (NE == 1 ? quad : 4 * quad + e);
        // (16 bits: what the second product's MFMA takes)
        if (i < count && p < a.I)
          reinterpret_cast<uint16_t*>(a.act)[static_cast<int64_t>(list[i]) * a.I + p] =
              lin_round16(decode_act(gate[e], up[e]), a.type);
      }
    }
    if constexpr (KS > 1) __syncthreads();
  }
}

// A single row: a wave takes one entry, R / 2 loads of gate rows and the up rows beside
// them.
template <class F, int L, int R, int DEPTH>
__global__ void __launch_bounds__(64 * kWaves) decode_up_single_kernel(const DecodeArgs a) {
  constexpr int RI = 64 / L, ROWS = R / 2 * RI, N = gemv_sums<L, R>();
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.I + kWaves * ROWS - 1) / (kWaves * ROWS);
  const int entry = blockIdx.x / tiles;
  const int i0 = ((blockIdx.x - entry * tiles) * kWaves + wave) * ROWS;
  if (i0 >= a.I) return;
  const int expert = __builtin_amdgcn_readfirstlane(decode_expert(a, entry));
  if (expert < 0) return;
  auto inner = [&](int r) { return i0 + r * RI < a.I - RI ? i0 + r * RI : a.I - RI; };
  float acc[R], sum[N];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.0f;
  gemv_add<F, L, R, DEPTH>(
      acc, a.up, expert, [&](int r) { return r < R / 2 ? inner(r) : a.I + inner(r - R / 2); }, a.x, a.H,
      0, gemv_chunks<F, L>(a.H));
  gemv_reduce<L, R>(acc, sum);
  uint16_t* act = reinterpret_cast<uint16_t*>(a.act) + static_cast<int64_t>(entry) * a.I;
#pragma unroll
  for (int q = 0; q < N / 2; ++q)
    if ((lane & 15) == q) {
      const int r = gemv_row<L>(q, lane >> 4);
      act[inner(r / RI) + r % RI] = lin_round16(decode_act(sum[q], sum[q + N / 2]), a.type);
    }
}

template <class F>
int launch_single(const DecodeArgs& a, hipStream_t s, const char* what) {
  constexpr int R = 8, DEPTH = F::dense ? 4 : 2;
  const int lanes = gemv_lanes<F>(a.H, a.I);
  const unsigned grid = static_cast<unsigned>(a.n * ceil_div(a.I, kWaves * R / 2 * (64 / lanes)));
  if (lanes == 64) decode_up_single_kernel<F, 64, R, DEPTH><<<grid, 64 * kWaves, 0, s>>>(a);
  else if (lanes == 32) decode_up_single_kernel<F, 32, R, DEPTH><<<grid, 64 * kWaves, 0, s>>>(a);
  else decode_up_single_kernel<F, 16, R, DEPTH><<<grid, 64 * kWaves, 0, s>>>(a);
  return check_launch(what);
}

template <class F, int NE, int KS>
int launch(const DecodeArgs& a, hipStream_t s, const char* what) {
  const int64_t grid = (a.n > a.E ? a.E : a.n) * ceil_div(a.I, 16 * (kWaves / KS)) + 1;
  MGQ_REQUIRE(grid < int64_t(1) << 24, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  decode_up_kernel<F, NE, KS, 2><<<static_cast<unsigned>(grid), 64 * kWaves, 0, s>>>(a);
  return check_launch(what);
}

}  // namespace

int decode_up(const DecodeArgs& a, int format, hipStream_t s, const char* what) {
  return decode_dispatch(format, a.type, a.up.type, [&](auto f) {
    using F = decltype(f);
    if (a.T == 1) return launch_single<F>(a, s, what);
    if (a.T <= 4) return launch<F, 1, 4>(a, s, what);
    return launch<F, 4, 2>(a, s, what);
  });
}

}  // namespace mgq
