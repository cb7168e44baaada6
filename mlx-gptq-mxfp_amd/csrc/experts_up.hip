// First launch of a routed layer for a few rows (experts_decode.h): gate and up
// projection of every entry and their activation, and the plan for the second launch.
//
// A workgroup takes 16 gate rows and the 16 up rows beside them of one expert, with all
// entries of that expert: its weight is read once (again for every further 16 entries).
// Only the device knows how many experts the rows have: a workgroup finds the slot-th of
// them in the list, which is short enough for every wave to look through, and those past
// the last one end there (they come last, where they hold up nobody).
//
// Up to 64 entries the four waves of a workgroup share the contraction, so that there are
// workgroups for every CU; beyond, each takes rows of its own and the lookup is paid by four
// times as many rows (64 rows of MXFP8, 128 experts of 2 x 768 x 2048: 102 us for 416 MB, 120
// with shared contractions; 16 rows of 4-bit codes: 25 against 37). The plan takes 8 us for
// 128 entries, the lookup 2 before the first load; the rest is steps (few_core.h) at 1 us for
// a wave alone, half of it waits for a step's codes, also when they are cached (vector
// instructions are 14 of the 102 us).
// One row: gemv_core.h, 11 us for 50 MB of bf16 and 5.7 us for 13 MB of MXFP4.
#include "experts_decode.h"

namespace mgq {
namespace {

// One workgroup of 256: the entries in the order (expert, place in the list), by counting
// for each how many come before it, and the items that they fall into. A row that names an
// expert twice is one entry with the sum of its weights. `keys` and `sorted` are LDS for
// kDecodeEntries each.
__device__ void decode_plan(const DecodeArgs& a, int32_t* keys, int32_t* sorted) {
  constexpr int kOwn = kDecodeEntries / 256;  // entries of a thread
  constexpr int32_t kNone = 0x7fffffff;
  const int tid = threadIdx.x, n4 = (a.n + 3) / 4;
  DecodeItem* items = reinterpret_cast<DecodeItem*>(a.plan + kDecodePlanHead / 4);
  DecodeEntry* entries = reinterpret_cast<DecodeEntry*>(items + a.n);
  int32_t key[kOwn];
  float weight[kOwn];
#pragma unroll
  for (int r = 0; r < kOwn; ++r) {
    const int i = tid + 256 * r;
    key[r] = i < a.n ? decode_expert(a, i) : -1;
    weight[r] = i < a.n ? a.weights[i] : 0.0f;
    keys[i] = key[r];
    sorted[i] = kNone;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kOwn; ++r) {
    const int i = tid + 256 * r, e = key[r];
    if (256 * r >= a.n || e < 0) {
      key[r] = kNone;
      continue;
    }
    bool again = false;
    const int row = i / a.k * a.k;
    for (int j = row; j < row + a.k; ++j)
      if (j != i && keys[j] == e) {
        again |= j < i;
        weight[r] += a.weights[j];
      }
    key[r] = again ? kNone : e * kDecodeEntries + i;  // (at most 2^20 experts)
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kOwn; ++r) keys[tid + 256 * r] = key[r];
  __syncthreads();
  int place[kOwn] = {};
  for (int j = 0; j < n4; ++j) {
    const int4 v = reinterpret_cast<const int4*>(keys)[j];
#pragma unroll
    for (int r = 0; r < kOwn; ++r)
      if (256 * r < a.n) place[r] += (v.x < key[r]) + (v.y < key[r]) + (v.z < key[r]) + (v.w < key[r]);
  }
#pragma unroll
  for (int r = 0; r < kOwn; ++r)
    if (key[r] != kNone) {
      sorted[place[r]] = key[r];
      entries[place[r]] = DecodeEntry{key[r] % kDecodeEntries, weight[r]};
    }
  for (int i = tid; i < a.tiles; i += 256) a.counts[i] = 0;
  __syncthreads();
  if (tid >= 64) return;
  // an item starts at every kDecodeItem-th entry of an expert
  int32_t* firsts = keys;
  int n_items = 0, total = 0, run = 0;
  for (int c = 0; c < a.n; c += 64) {
    const int p = c + tid;
    const int32_t v = p < a.n ? sorted[p] : kNone;
    const int expert = v / kDecodeEntries;
    const uint64_t upto = ~uint64_t(0) >> (63 - tid);
    const uint64_t starts = __ballot(v != kNone && (p == 0 || sorted[p - 1] / kDecodeEntries != expert));
    const uint64_t before = starts & upto;
    const int start = before ? c + 63 - __builtin_clzll(before) : run;
    const bool opens = v != kNone && (p - start) % kDecodeItem == 0;
    const uint64_t open = __ballot(opens);
    if (opens) {
      const int item = n_items + __popcll(open & (upto >> 1));
      firsts[item] = p;
      items[item].expert = expert;
    }
    n_items += __popcll(open);
    total += __popcll(__ballot(v != kNone));
    if (starts) run = c + 63 - __builtin_clzll(starts);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int i = tid; i < n_items; i += 64) {
    const int first = firsts[i], end = i + 1 < n_items ? firsts[i + 1] : total;
    items[i].first = static_cast<uint16_t>(first);
    items[i].count = static_cast<uint16_t>(end - first);
  }
  if (tid == 0) a.plan[0] = n_items;
}

constexpr int kWaves = 4;

__device__ __forceinline__ float decode_act(float gate, float up) {
  return gate / (1.0f + expf(-gate)) * up;
}

constexpr int kTable = kDecodeEntries;  // experts whose first entries LDS holds

// KS waves share the contraction; the others take 16 gate rows each.
template <class F, int NE, int KS, int DEPTH>
__global__ void __launch_bounds__(64 * kWaves) decode_up_kernel(const DecodeArgs a) {
  constexpr int BM = NE == 1 ? 4 : 16, BP = 16 * (kWaves / KS);
  // (the plan's keys and their order; the list of the workgroup's entries and the table)
  __shared__ __attribute__((aligned(16))) int32_t list[kDecodeEntries], first_of[kTable];
  __shared__ lin_f32x4_t part[KS > 1 ? kWaves * 2 * 64 : 1];
  __shared__ __attribute__((aligned(16))) char params[F::dense ? 16 : kWaves * few_lds<F, 2>()];
  if (blockIdx.x == 0) {
    decode_plan(a, list, first_of);
    return;
  }
  const int bid = blockIdx.x - 1;
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (a.I + BP - 1) / BP, kw = wave % KS;
  const int slot = bid / tiles, p0 = (bid - slot * tiles) * BP + wave / KS * 16, p = p0 + r16;
  // The list goes through registers, in halves of a fixed size that most calls need one of.
  constexpr int kChunks = 8;
  const int halves = (a.n + 64 * kChunks - 1) / (64 * kChunks);
  int ids[kChunks];
  auto load_ids = [&](int half) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int i = 64 * (kChunks * half + c) + lane;
      ids[c] = -1;
      if (64 * (kChunks * half + c) < a.n && i < a.n) ids[c] = decode_expert(a, i);
    }
  };
  // f(chunk of ids, first place) for the chunks there are
  auto chunks = [&](auto&& f) {
    for (int half = 0; half < halves; ++half) {
      if (halves > 1) load_ids(half);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int i0 = 64 * (kChunks * half + c);
        if (i0 >= a.n) break;
        f(ids[c], i0);
      }
    }
  };
  const uint64_t below = (uint64_t(1) << lane) - 1;
  if (halves == 1) load_ids(0);
  // this workgroup's expert
  int expert = -1;
  if (a.E <= kTable) {
    // the slot-th entry that is its expert's first one
    for (int i = threadIdx.x; i < a.E; i += 64 * kWaves) first_of[i] = kDecodeEntries;
    __syncthreads();
    chunks([&](int id, int i0) {
      if (i0 / 64 % kWaves == wave && id >= 0) atomicMin(first_of + id, i0 + lane);
    });
    __syncthreads();
    int seen = 0;
    chunks([&](int id, int i0) {
      const bool leads = id >= 0 && first_of[id] == i0 + lane;
      const uint64_t mask = __ballot(leads);
      const uint64_t hit = __ballot(leads && seen + __popcll(mask & below) == slot);
      if (hit) expert = __builtin_amdgcn_readlane(id, __builtin_ctzll(hit));
      seen += __popcll(mask);
    });
  } else {
    // entry `slot`'s, if no entry before it has the same one
    const int mine = __builtin_amdgcn_readfirstlane(decode_expert(a, slot));
    bool earlier = mine < 0;
    chunks([&](int id, int i0) { earlier |= __ballot(id == mine && i0 + lane < slot) != 0; });
    if (!earlier) expert = mine;
  }
  if (expert < 0) return;
  int count = 0;
  chunks([&](int id, int i0) {
    const uint64_t mask = __ballot(id == expert);
    if (wave == 0 && id == expert) list[count + __popcll(mask & below)] = i0 + lane;
    count += __popcll(mask);
  });
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
        if (i < count && p < a.I) decode_store_act(a, list[i], p, decode_act(gate[e], up[e]));
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
#pragma unroll
  for (int q = 0; q < N / 2; ++q)
    if ((lane & 15) == q) {
      const int r = gemv_row<L>(q, lane >> 4);
      decode_store_act(a, entry, inner(r / RI) + r % RI, decode_act(sum[q], sum[q + N / 2]));
    }
}

template <class F>
int launch_single(const DecodeArgs& a, hipStream_t s, const char* what) {
  constexpr int R = 8, DEPTH = F::dense ? 4 : 2;
  const int lanes = gemv_lanes<F>(a.H, a.I);
  const int64_t blocks = a.n * ceil_div(a.I, kWaves * R / 2 * (64 / lanes));
  MGQ_REQUIRE(blocks < int64_t(1) << 24, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  const unsigned grid = static_cast<unsigned>(blocks);
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
    return a.n <= 64 ? launch<F, 4, 4>(a, s, what) : launch<F, 4, 1>(a, s, what);
  });
}

}  // namespace mgq
