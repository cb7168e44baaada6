// Products of few rows: a group has a handful of list entries (single tokens,
// small decoding batches), so the weight is read once and reading it is the
// work.
//
// A workgroup computes 16 NQ entries x 16 NP weight rows; its waves share the
// contraction and add their sums through LDS in wave order. The weight goes from
// memory into registers as the A operand of a 16x16 MFMA (lane l: row l % 16, a
// 16-byte piece of it by l / 16), X from the caches as its B operand; nothing is
// staged, so a wave has all the loads of a batch in flight at once. Any pitch
// and alignment: a 16-byte load takes any address, and the pieces in which a row
// ends are read element by element.
//
// An MX weight's lane reads the 32 codes of one group and its scale byte; the
// four quarters of a wave take four consecutive groups, so MFMA i of four
// multiplies codes 8 i .. 8 i + 7 of each.
//
// Measured, called again on the same weights (the 256 MB memory-side cache holds them):
// one token through 8 of 128 experts [1536, 2048], bf16 11 us (4.6 TB/s of weight), MXFP4
// codes 8 us, of which a launch with its two dependent loads (offsets, row index) takes 5;
// one row of bf16 [14336, 4096] 22 us, and 44 us (2.7 TB/s) after 512 MiB were written
// elsewhere. One row of int8 of that shape takes 12.6 us here (24.5 after the writes); the
// time model prices it as 19 us and gives it to the 64 x 128 tile, which takes 15.0 (27.1).
// A group's second 16 entries repeat its weight from L2; 64 entries in one workgroup
// (NQ = 4) load it once.
#include "linear_few.h"

namespace mgq {
namespace {

// The 16 bytes at `at` of a row whose pieces may end inside it, zeros for what
// is past its end.
template <int ES>
__device__ __forceinline__ lin_u32x4_t cut_piece(const char* row, int64_t at, int64_t row_bytes) {
  lin_u32x4_t r = {0, 0, 0, 0};
  if (at + 16 <= row_bytes) {
    const lin_u128_u_t u = *reinterpret_cast<const lin_u128_u_t*>(row + at);
    r = lin_u32x4_t{u.v[0], u.v[1], u.v[2], u.v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i)
      if (at + i * ES < row_bytes) {
        const uint32_t v = ES == 2 ? *reinterpret_cast<const uint16_t*>(row + at + 2 * i)
                                   : *reinterpret_cast<const uint8_t*>(row + at + i);
        r[i * ES / 4] |= v << (8 * ((i * ES) & 3));
      }
  }
  return r;
}
// A piece that is known to lie inside its row.
template <bool AL>
__device__ __forceinline__ lin_u32x4_t whole_piece(const char* at) {
  if constexpr (AL) return *reinterpret_cast<const lin_u32x4_t*>(at);
  const lin_u128_u_t u = *reinterpret_cast<const lin_u128_u_t*>(at);
  return lin_u32x4_t{u.v[0], u.v[1], u.v[2], u.v[3]};
}

template <int OP>
__device__ __forceinline__ typename LinAcc<OP>::t16 mfma16(lin_u32x4_t a, lin_u32x4_t b,
                                                           typename LinAcc<OP>::t16 c) {
  if constexpr (OP == kOpI8)
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(lin_i32x4_t, a),
                                                 __builtin_bit_cast(lin_i32x4_t, b), c, 0, 0, 0);
  else if constexpr (OP == kOpF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lin_f16x8_t, a),
                                                  __builtin_bit_cast(lin_f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lin_bf16x8_t, a),
                                                   __builtin_bit_cast(lin_bf16x8_t, b), c, 0, 0, 0);
}

// Waves that share the contraction. Two and eight measured the same within 10 % for
// 16-bit weights, eight up to twice slower for MXFP4 (too few codes a wave).
constexpr int kWaves = 4;

template <int OP, int NP, int NQ, bool AL>
__global__ void __launch_bounds__(64 * kWaves) lin_few_kernel(const LinArgs a) {
  constexpr int ES = lin_esize<OP>();
  constexpr bool MX = lin_is_mx<OP>();
  constexpr int STEP = MX ? 256 : 64;        // bytes of an X row per step
  // steps loaded at once
  constexpr int BATCH = OP == kOpMx4 ? (NQ > 1 ? 2 : 4) : OP == kOpMx8 ? (NQ > 2 ? 1 : 2)
                                                                     : (NQ > 2 ? 4 : 8);
  constexpr int CB = OP == kOpMx4 ? 16 : 32;                      // MX: bytes of a group's codes
  constexpr int WV = MX ? CB / 16 : 1, XV = MX ? 4 : 1;           // 16-byte loads per step
  typedef typename LinAcc<OP>::t16 acc_t;
  __shared__ acc_t part[kWaves * NP * NQ * 64];

  LinTile t;
  if (!lin_find_tile<16 * NQ>(a, (a.np + 16 * NP - 1) / (16 * NP), &t)) return;
  const int lane = threadIdx.x & 63, r16 = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int waves = kWaves;
  const int g = t.g, gw = g < a.G ? g : 0;
  const int p0 = t.pt * 16 * NP;
  const int64_t row_bytes = static_cast<int64_t>(a.nc) * ES;
  const int steps = g < a.G ? static_cast<int>((row_bytes + STEP - 1) / STEP) : 0;
  const int full = static_cast<int>(row_bytes / STEP);  // steps with every piece inside the row
  // this wave's steps, an even number so that it reads whole 128-byte lines
  constexpr int EVEN = MX ? ~0 : ~1;
  const int s_begin = static_cast<int>(static_cast<int64_t>(steps) * wave / waves) & EVEN;
  const int s_end = wave + 1 == waves
                        ? steps
                        : static_cast<int>(static_cast<int64_t>(steps) * (wave + 1) / waves) & EVEN;

  const char* w[NP];
  const uint8_t* ws[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    int p = p0 + 16 * i + r16;
    p = p < a.np ? p : a.np - 1;
    w[i] = a.P + gw * a.p_group + p * a.ldp;
    ws[i] = MX ? a.Ps + (static_cast<int64_t>(gw) * a.np + p) * (a.nc / 32) : nullptr;
  }
  acc_t acc[NP][NQ];
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0;

  // One batch of weight loads is in flight beyond the batch being multiplied, and
  // the first one before the row of X is known (its index is a load of its own).
  // Steps past the end load the row's first piece and are cleared when they are
  // multiplied, so that no load is waited for before its use.
  lin_u32x4_t wv[2][BATCH][NP][WV], xv[BATCH][NQ][XV];
  uint32_t sc[2][BATCH][NP];
  constexpr int PIECE = MX ? 64 : 16;  // X bytes of a lane and step
  const int64_t x_lane = quad * PIECE;
  auto inside = [&](int st) {  // this lane's part of the step is inside the row
    return st < s_end && st * static_cast<int64_t>(STEP) + x_lane < row_bytes;
  };
  auto whole = [&](int s) { return s + BATCH <= full && s + BATCH <= s_end; };
  auto load_w = [&](int k, int s) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const bool ok = inside(s + b);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (MX) {
          const int64_t at = ok ? static_cast<int64_t>(s + b) * 4 * CB + quad * CB : 0;
#pragma unroll
          for (int v = 0; v < WV; ++v) wv[k][b][i][v] = whole_piece<AL>(w[i] + at + 16 * v);
          sc[k][b][i] = ws[i][ok ? 4 * (s + b) + quad : 0];
        } else if constexpr (AL) {
          wv[k][b][i][0] =
              whole_piece<AL>(w[i] + (ok ? static_cast<int64_t>(s + b) * STEP + quad * 16 : 0));
        }
      }
    }
    if constexpr (!MX && !AL) {
      if (whole(s)) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
          for (int i = 0; i < NP; ++i)
            wv[k][b][i][0] = whole_piece<AL>(w[i] + static_cast<int64_t>(s + b) * STEP + quad * 16);
      } else {
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
#pragma unroll
          for (int i = 0; i < NP; ++i)
            wv[k][b][i][0] = cut_piece<ES>(
                w[i], s + b < s_end ? static_cast<int64_t>(s + b) * STEP + quad * 16 : row_bytes,
                row_bytes);
      }
    }
  };
  if (s_begin < s_end) load_w(0, s_begin);

  const char* x[NQ];
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    const int64_t q = t.q0 + 16 * j + r16;
    x[j] = a.Q + lin_row(a, q < t.q_end ? q : t.q_end - 1) * a.ldq;
  }
  auto load_x = [&](int s) {
    if constexpr (MX || AL) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int64_t at = inside(s + b) ? static_cast<int64_t>(s + b) * STEP + x_lane : 0;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int v = 0; v < XV; ++v) xv[b][j][v] = whole_piece<AL>(x[j] + at + 16 * v);
      }
    } else if (whole(s)) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
          xv[b][j][0] = whole_piece<AL>(x[j] + static_cast<int64_t>(s + b) * STEP + quad * 16);
    } else {
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
          xv[b][j][0] = cut_piece<ES>(
              x[j], s + b < s_end ? static_cast<int64_t>(s + b) * STEP + quad * 16 : row_bytes,
              row_bytes);
    }
  };
  auto multiply = [&](int k, int s) {
    if ((MX || AL) && !whole(s)) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const uint32_t keep = inside(s + b) ? 0xffffffffu : 0u;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int v = 0; v < XV; ++v) xv[b][j][v] &= keep;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
#pragma unroll
          for (int v = 0; v < WV; ++v) wv[k][b][i][v] &= keep;
          if constexpr (MX) sc[k][b][i] &= keep;
        }
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
#pragma unroll
      for (int v = 0; v < XV; ++v)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          lin_u32x4_t m = wv[k][b][i][0];
          if constexpr (OP == kOpMx4)
            m = lin_decode_mx4(wv[k][b][i][0][v], sc[k][b][i]);
          else if constexpr (OP == kOpMx8)
            m = lin_decode_mx8(wv[k][b][i][v >> 1][2 * (v & 1)],
                               wv[k][b][i][v >> 1][2 * (v & 1) + 1], sc[k][b][i]);
#pragma unroll
          for (int j = 0; j < NQ; ++j) acc[i][j] = mfma16<OP>(m, xv[b][j][v], acc[i][j]);
        }
  };
  for (int s = s_begin; s < s_end; s += 2 * BATCH) {
    load_x(s);
    if (s + BATCH < s_end) load_w(1, s + BATCH);
    multiply(0, s);
    if (s + BATCH >= s_end) break;
    load_x(s + BATCH);
    if (s + 2 * BATCH < s_end) load_w(0, s + 2 * BATCH);
    multiply(1, s + BATCH);
  }

#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) part[((wave * NP + i) * NQ + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  // block (i, j) of the tile is summed and stored by wave (i NQ + j) % waves
  for (int blk = wave; blk < NP * NQ; blk += waves) {
    acc_t sum = part[blk * 64 + lane];
    for (int o = 1; o < waves; ++o) {
      const acc_t v = part[(o * NP * NQ + blk) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
    const int p = p0 + 16 * (blk / NQ) + 4 * quad;
    const int64_t q = t.q0 + 16 * (blk % NQ) + r16;
    if (q >= t.q_end || p >= a.np) continue;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(sum[e]);
    if constexpr (OP == kOpI8) {
      if (g < a.G) lin_scale4<OP>(a, g, p, a.sx[lin_row(a, q)], v);
    }
    lin_store4(a, a.out + q * a.ldo * (a.out_type == kF32 ? 4 : 2), p, v);
  }
}

template <int OP, int NQ>
int launch(const LinArgs& a, hipStream_t s, const char* what) {
  constexpr int NP = NQ == 4 ? 2 : 1;  // lin_few_cols(NQ) / 16
  const int64_t grid = lin_few_grid(a, NQ);
  MGQ_REQUIRE(grid < kLinFewGrid, MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  if ((lin_row_bounds(a, static_cast<int64_t>(a.nc) * lin_esize<OP>()) & 15) == 0)
    lin_few_kernel<OP, NP, NQ, true><<<static_cast<unsigned>(grid), 64 * kWaves, 0, s>>>(a);
  else
    lin_few_kernel<OP, NP, NQ, false><<<static_cast<unsigned>(grid), 64 * kWaves, 0, s>>>(a);
  return check_launch(what);
}

template <int OP>
int run(const LinArgs& a, int nq, hipStream_t s, const char* what) {
  if (nq == 1) return launch<OP, 1>(a, s, what);
  if (nq == 2) return launch<OP, 2>(a, s, what);
  return launch<OP, 4>(a, s, what);
}

}  // namespace

int lin_few_rows(const LinArgs& a, int op, int nq, hipStream_t s, const char* what) {
  switch (op) {
    case kOpBF16: return run<kOpBF16>(a, nq, s, what);
    case kOpF16: return run<kOpF16>(a, nq, s, what);
    case kOpI8: return run<kOpI8>(a, nq, s, what);
    case kOpMx4: return run<kOpMx4>(a, nq, s, what);
    default: return run<kOpMx8>(a, nq, s, what);
  }
}

}  // namespace mgq
