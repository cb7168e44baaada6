// Large tiles of the matrix products, for operands whose rows start and end on
// 16-byte boundaries (linear_common.h has the products and their operands).
//
// Tile kernel: 512 threads = 8 waves, 2 along q and 4 along p, one workgroup
// per CU. A wave owns 32 FQ x 64 outputs as FQ x 2 blocks of a 32x32 MFMA (at
// FQ = 4 a 256 x 256 tile, 128 fp32 accumulators per lane).
//
//   - A stage is 128 bytes of every row: 64 16-bit or 128 int8 elements of the
//     contraction, four K-steps of one MFMA depth each. The rows go from memory
//     straight into LDS (global_load_lds_dwordx4, 16 bytes a lane), NB stages
//     deep. What lies past the contraction's end reads a page of zeros; rows past
//     the operand's end repeat its last row and their results are not stored.
//   - Plain operands keep 128-byte rows in LDS. The 16-byte chunk c of row r
//     sits at c ^ (r / 2 % 8): the lanes of an MFMA operand read the same chunk of
//     32 consecutive rows, and any 16 of them cover all 64 banks once.
//   - Transposed operands keep contraction rows (64 of them) in LDS as they are
//     in memory; ds_read_b64_tr_b16 hands a lane one column of four rows. The
//     64-byte block b of row t sits at b ^ (t % 4).
//   - An MX weight's codes stay codes in LDS (32 or 64 bytes a row and stage, and
//     its two scale bytes widened to dwords). Half-wave h of the MFMA takes the
//     stage's elements 32 h .. 32 h + 31, one MX group, so a lane needs one scale
//     a stage and its codes in one or two 16-byte reads; they are decoded to bf16
//     in registers, two a conversion, 8 conversions beside 8 MFMAs.
//   - K-step schedule: each MFMA is followed by its share of the next K-step's
//     LDS reads, and in the first K-step after a stage's barrier by the loads of
//     the stage that takes the buffer just released. The last K-step of a stage
//     runs after the barrier, over the first reads of the next stage.
#include "linear_tile.h"

namespace mgq {
namespace {

constexpr int kBP = 256;
constexpr int kRowB = 128;  // bytes of a plain row per stage
constexpr int kLdsMax = 160 * 1024;

__device__ uint32_t g_lin_zeros[64];  // never written: what lies past an operand's end

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) lin_u32x4_t lds_u32x4;
typedef short lin_s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lin_s16x4_t lds_s16x4;
typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;

// Wait until at most VM of this wave's loads are in flight and its LDS reads are
// done, then for the other waves. The memory clobber orders the LDS accesses for
// the compiler as __syncthreads would, without its wait for every load.
template <int VM>
__device__ __forceinline__ void stage_barrier() {
  static_assert(VM <= 63, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
}

// 16 bytes (1 byte, widened to a dword) per lane from `src` to LDS at
// dst + 16 (4) * lane.
__device__ __forceinline__ void dma16(uint32_t dst, uint64_t src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
__device__ __forceinline__ void dma1(uint32_t dst, uint64_t src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(dst), "v"(src) : "memory");
}

__device__ __forceinline__ lin_u32x4_t read16(uint32_t at) {
  return *reinterpret_cast<const lds_u32x4*>(at);
}
// Eight contraction rows of a lane's column: rows 0..3 at `at`, 4..7 below.
__device__ __forceinline__ lin_u32x4_t read_tr(uint32_t at, int pitch) {
  const lin_s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at));
  const lin_s16x4_t hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4*>(at + 4 * pitch));
  const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
  return lin_u32x4_t{l.x, l.y, h.x, h.y};
}

template <int OP>
constexpr int p_stage_bytes() {
  return OP == kOpMx4 ? kBP * 32 + kBP * 8 : OP == kOpMx8 ? kBP * 64 + kBP * 8 : kBP * kRowB;
}
template <int OP, int FQ>
constexpr int n_buffers() {
  const int n = kLdsMax / (64 * FQ * kRowB + p_stage_bytes<OP>());
  return n > 4 ? 4 : n;
}

template <int OP, int KIND, int FQ>
__global__ void __launch_bounds__(512, 1) lin_tile_kernel(const LinArgs a, const LinPlanArgs pl) {
  constexpr bool PT = KIND != kLinForward;
  constexpr bool QT = KIND == kLinWgrad;
  constexpr bool MX = lin_is_mx<OP>();
  constexpr int ES = lin_esize<OP>();
  constexpr int BQ = 64 * FQ;
  constexpr int QB = BQ * kRowB;                 // Q bytes per stage
  constexpr int SB = QB + p_stage_bytes<OP>();   // stage bytes
  constexpr int NB = n_buffers<OP, FQ>();
  constexpr int EPI = BQ * kBP * 2;              // 16-bit results on their way out
  constexpr int VQ = FQ;                         // loads per wave and stage
  constexpr int VP = OP == kOpMx4 ? 2 : OP == kOpMx8 ? 3 : 4;
  constexpr int V = VQ + VP;
  constexpr int NM = 2 * FQ;                     // MFMAs per K-step
  constexpr int EK = kRowB / ES;                 // contraction elements per stage
  static_assert(NB >= 2 && (NB - 2) * V <= 63, "stages");
  static_assert(!QT || FQ == 4, "transposed Q tiles are 256 wide");
  __shared__ __attribute__((aligned(1024))) char lds[NB * SB > EPI ? NB * SB : EPI];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wq = wave >> 2, wp = wave & 3;
  const int half = lane >> 5;

  // ---- which tile -------------------------------------------------------
  int g, p0, slot = -1;
  int64_t q0, q_end;                 // rows of Q (forward, dgrad) or of the output (wgrad)
  int64_t c_begin = 0, c_len = a.nc;  // contraction range
  if constexpr (KIND == kLinWgrad) {
    LinUnit u;
    int tile;
    if (!lin_find_unit(a, pl, &u, &tile)) return;
    g = u.g;
    slot = u.slot;
    c_begin = u.t0;
    c_len = u.t1 - u.t0;
    q0 = static_cast<int64_t>(tile % pl.nqt) * BQ;
    p0 = tile / pl.nqt * kBP;
    q_end = a.nq;
  } else {
    LinTile t;
    if (!lin_find_tile<BQ>(a, (a.np + kBP - 1) / kBP, &t)) return;
    g = t.g;
    p0 = t.pt * kBP;
    q0 = t.q0;
    q_end = t.q_end;
    if (g >= a.G) c_len = 0;  // entries of no group: zeros
  }
  const int gw = KIND == kLinWgrad || g >= a.G ? 0 : g;
  const char* Pg = a.P + gw * a.p_group;
  const int n_stages = static_cast<int>((c_len + EK - 1) / EK);

  // ---- loads ------------------------------------------------------------
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char*)lds));
  const uint64_t zeros = reinterpret_cast<uint64_t>(g_lin_zeros);
  // plain rows: instruction i of a wave takes rows 8 (n wave + i) .. + 7, lane l
  // the chunk l % 8 of row l / 8, which holds the row's chunk ^ its swizzle
  // (that depends on i's parity only)
  const int ch0 = (lane & 7) ^ ((lane >> 4) & 7), ch1 = ch0 ^ 4;
  // transposed rows: instruction i takes contraction rows 8 wave + 2 i, + 1
  const int tr_row = 8 * wave + half;
  const int tc0 = (lane & 31) ^ (4 * half), tc1 = tc0 ^ 8;
  uint64_t qp[VQ], pp[MX ? VP : 4];
  if constexpr (QT) {
#pragma unroll
    for (int i = 0; i < VQ; ++i) {
      int64_t col = q0 + 8 * (i & 1 ? tc1 : tc0);
      col = col + 8 <= a.nq ? col : a.nq - 8;
      qp[i] = reinterpret_cast<uint64_t>(a.Q) + (c_begin + tr_row + 2 * i) * a.ldq + 2 * col;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VQ; ++i) {
      int64_t q = q0 + 8 * (VQ * wave + i) + (lane >> 3);
      q = q < q_end ? q : q_end - 1;
      const int64_t row = KIND == kLinForward ? lin_row(a, q) : q;
      const int sw = ((VQ * wave + i) & 1) ? ch1 : ch0;
      qp[i] = reinterpret_cast<uint64_t>(a.Q) + row * a.ldq + 16 * sw;
    }
  }
  const uint8_t* Psg = nullptr;
  if constexpr (MX) {
    Psg = a.Ps + static_cast<int64_t>(gw) * a.np * (a.nc / 32);
    constexpr int per = OP == kOpMx4 ? 2 : 4;  // 16-byte pieces of a row's codes
#pragma unroll
    for (int i = 0; i < VP - 1; ++i) {
      const int r = 32 * wave + (64 / per) * i + lane / per;
      const int pos = lane % per;
      const int c = per == 2 ? pos ^ ((r >> 3) & 1) : pos ^ ((r >> 2) & 3);
      const int p = p0 + r < a.np ? p0 + r : a.np - 1;
      pp[i] = reinterpret_cast<uint64_t>(Pg) + p * a.ldp + 16 * c;
    }
    const int r = 32 * wave + (lane >> 1);
    const int p = p0 + r < a.np ? p0 + r : a.np - 1;
    pp[VP - 1] = reinterpret_cast<uint64_t>(Psg) + static_cast<int64_t>(p) * (a.nc / 32) + (lane & 1);
  } else if constexpr (PT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int64_t col = p0 + 8 * (i & 1 ? tc1 : tc0);
      col = col + 8 <= a.np ? col : a.np - 8;
      // wgrad: the row is added when it is known
      pp[i] = reinterpret_cast<uint64_t>(Pg) + 2 * col +
              (KIND == kLinWgrad ? 0 : (tr_row + 2 * i) * a.ldp);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * (4 * wave + i) + (lane >> 3);
      const int p = p0 + r < a.np ? p0 + r : a.np - 1;
      pp[i] = reinterpret_cast<uint64_t>(Pg) + p * a.ldp + 16 * (i & 1 ? ch1 : ch0);
    }
  }

  // wgrad: the rows of X that this wave loads in the next stage, two per
  // instruction, read through the scalar cache (a vector load's wait would also
  // wait for the loads into LDS before it)
  uint32_t rows[8];
  auto load_rows = [&](int st) {
    if constexpr (KIND == kLinWgrad) {
      const int64_t t0 = c_begin + static_cast<int64_t>(st) * EK + 8 * wave;
      const int64_t last = c_begin + c_len - 1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t t = t0 + i < last ? t0 + i : last;
        int32_t r = static_cast<int32_t>(t);
        if (a.row_index) {
          r = reinterpret_cast<const_i32_ptr>(reinterpret_cast<uint64_t>(a.row_index))[t];
          r = r < 0 ? 0 : r;
          r = r < a.n_rows ? r : static_cast<int32_t>(a.n_rows - 1);
        }
        rows[i] = static_cast<uint32_t>(r);
      }
    }
  };

  // load i of stage st into buffer at LDS address `buf`
  auto load = [&](int i, int st, uint32_t buf) {
    if (i < VQ) {
      bool ok;
      if constexpr (QT) {
        ok = tr_row + 2 * i < c_len - static_cast<int64_t>(st) * EK;
      } else {
        const int64_t rem = (c_len - static_cast<int64_t>(st) * EK) * ES;
        ok = 16 * (((VQ * wave + i) & 1) ? ch1 : ch0) < rem;
      }
      dma16(buf + (VQ * wave + i) * 1024, ok ? qp[i] : zeros);
      qp[i] += QT ? EK * a.ldq : kRowB;
      return;
    }
    const int k = i - VQ;
    if constexpr (MX) {
      const int64_t rem = c_len / 32 - 2 * static_cast<int64_t>(st);  // MX groups left
      constexpr int per = OP == kOpMx4 ? 2 : 4;
      if (k < VP - 1) {
        const int r = 32 * wave + (64 / per) * k + lane / per;
        const int pos = lane % per;
        const int c = per == 2 ? pos ^ ((r >> 3) & 1) : pos ^ ((r >> 2) & 3);
        dma16(buf + QB + ((VP - 1) * wave + k) * 1024, (c * 2 / per) < rem ? pp[k] : zeros);
        pp[k] += 16 * per;
      } else {
        dma1(buf + QB + kBP * 16 * per + wave * 256, (lane & 1) < rem ? pp[k] : zeros);
        pp[k] += 2;
      }
    } else if constexpr (PT) {
      const bool ok = tr_row + 2 * k < c_len - static_cast<int64_t>(st) * EK;
      uint64_t src = pp[k];
      if constexpr (KIND == kLinWgrad) {
        const uint32_t r = half ? rows[2 * k + 1] : rows[2 * k];
        src += static_cast<uint64_t>(r) * static_cast<uint32_t>(a.ldp);
      } else {
        pp[k] += EK * a.ldp;
      }
      dma16(buf + QB + (4 * wave + k) * 1024, ok ? src : zeros);
    } else {
      const int64_t rem = (c_len - static_cast<int64_t>(st) * EK) * ES;
      dma16(buf + QB + (4 * wave + k) * 1024, 16 * (k & 1 ? ch1 : ch0) < rem ? pp[k] : zeros);
      pp[k] += kRowB;
    }
  };

  // ---- LDS reads of a K-step's operands -----------------------------------
  // plain: chunk 2 ks + half of the row (MX: 4 half + ks, so that a half-wave
  // keeps to its MX group)
  const int sw = (lane >> 1) & 7;
  uint32_t qa[4], pa[4];  // plain: by ks; transposed: by block
  const int j4 = (lane >> 2) & 3;
  const uint32_t tr_lane = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t c = 16 * ((MX ? 4 * half + k : 2 * k + half) ^ sw);
    qa[k] = QT ? (8 * half + j4) * (2 * BQ) + (((FQ * wq + k) ^ j4) * 64) + tr_lane
               : (32 * FQ * wq + (lane & 31)) * kRowB + c;
    pa[k] = PT ? QB + (8 * half + j4) * (2 * kBP) + (((2 * wp + (k & 1)) ^ j4) * 64) + tr_lane
               : QB + (64 * wp + (lane & 31)) * kRowB + c;
  }
  uint32_t code_at[2], scale_at = 0;
  if constexpr (MX) {
    constexpr int per = OP == kOpMx4 ? 2 : 4;
    const int r = 64 * wp + (lane & 31);
#pragma unroll
    for (int k = 0; k < per / 2; ++k) {
      const int c = per == 2 ? half : 2 * half + k;
      const int pos = per == 2 ? c ^ ((r >> 3) & 1) : c ^ ((r >> 2) & 3);
      code_at[k] = QB + r * 16 * per + 16 * pos;
    }
    scale_at = QB + kBP * 16 * per + (2 * r + half) * 4;
  }
  lin_u32x4_t fq[2][FQ], fp[2][2];
  lin_u32x4_t codes[2][2];
  uint32_t scale[2];
  auto read_q = [&](int b, int f, int ks, uint32_t buf) {
    if constexpr (QT)
      fq[b][f] = read_tr(buf + qa[f] + 16 * ks * (2 * BQ), 2 * BQ);
    else
      fq[b][f] = read16(buf + qa[ks] + f * 32 * kRowB);
  };
  auto read_p = [&](int b, int f, int ks, uint32_t buf) {
    if constexpr (PT)
      fp[b][f] = read_tr(buf + pa[f] + 16 * ks * (2 * kBP), 2 * kBP);
    else
      fp[b][f] = read16(buf + pa[ks] + f * 32 * kRowB);
  };
  auto read_codes = [&](int f, uint32_t buf) {
    constexpr int per = OP == kOpMx4 ? 2 : 4;
#pragma unroll
    for (int k = 0; k < per / 2; ++k) codes[f][k] = read16(buf + code_at[k] + f * 32 * 16 * per);
    scale[f] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(
        buf + scale_at + f * 32 * 8);
  };
  auto decode = [&](int b, int f, int ks) {
    if constexpr (OP == kOpMx4)
      fp[b][f] = lin_decode_mx4(codes[f][0][ks], scale[f]);
    else if constexpr (OP == kOpMx8)
      fp[b][f] = lin_decode_mx8(codes[f][ks >> 1][2 * (ks & 1)], codes[f][ks >> 1][2 * (ks & 1) + 1],
                                scale[f]);
  };
  // read r of a K-step (dense: p0 q0 p1 q1 q2 q3; MX: the q only)
  constexpr int NR = MX ? FQ : FQ + 2;
  auto read = [&](int r, int b, int ks, uint32_t buf) {
    if constexpr (MX) {
      read_q(b, r, ks, buf);
    } else if constexpr (FQ == 1) {
      if (r == 1) read_q(b, 0, ks, buf);
      else read_p(b, r >> 1, ks, buf);
    } else {
      if (r == 0) read_p(b, 0, ks, buf);
      else if (r == 2) read_p(b, 1, ks, buf);
      else read_q(b, r == 1 ? 0 : r - 2, ks, buf);
    }
  };

  typedef typename LinAcc<OP>::t32 acc_t;
  acc_t acc[FQ][2];
#pragma unroll
  for (int i = 0; i < FQ; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  if (n_stages > 0) {
#pragma unroll
    for (int st = 0; st < NB - 1; ++st) {
      load_rows(st);
#pragma unroll
      for (int i = 0; i < V; ++i) load(i, st, lds0 + st * SB);
    }
    load_rows(NB - 1);
    stage_barrier<(NB - 2) * V>();
    if constexpr (MX) {
      read_codes(0, lds0);
      read_codes(1, lds0);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) read(r, 0, 0, lds0);
#pragma unroll
    for (int i = 0; i < V; ++i) load(i, NB - 1, lds0 + (NB - 1) * SB);
    load_rows(NB);
    if constexpr (MX) {
      decode(0, 0, 0);
      decode(0, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    int rb = 0;
    for (int s = 0; s < n_stages; ++s) {
      const uint32_t buf = lds0 + rb * SB;
#pragma unroll
      for (int ks = 1; ks < 4; ++ks) {
        const int b = (ks - 1) & 1;
#pragma unroll
        for (int j = 0; j < NM; ++j) {
          acc[j >> 1][j & 1] = lin_mfma32<OP>(fp[b][j & 1], fq[b][j >> 1], acc[j >> 1][j & 1]);
#pragma unroll
          for (int r = j * NR / NM; r < (j + 1) * NR / NM; ++r) read(r, b ^ 1, ks, buf);
          if constexpr (MX) {
            if (j == 0) decode(b ^ 1, 0, ks);
            if (j == NM / 2) decode(b ^ 1, 1, ks);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (s + 1 == n_stages) break;
      rb = rb + 1 == NB ? 0 : rb + 1;
      const uint32_t next = lds0 + rb * SB;
      stage_barrier<(NB - 2) * V>();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MX) {
        read_codes(0, next);
        read_codes(1, next);
      }
#pragma unroll
      for (int j = 0; j < NM; ++j) {
        acc[j >> 1][j & 1] = lin_mfma32<OP>(fp[1][j & 1], fq[1][j >> 1], acc[j >> 1][j & 1]);
#pragma unroll
        for (int r = j * NR / NM; r < (j + 1) * NR / NM; ++r) read(r, 0, 0, next);
#pragma unroll
        for (int i = j * V / NM; i < (j + 1) * V / NM; ++i) load(i, s + NB, buf);
        __builtin_amdgcn_sched_barrier(0);
      }
      load_rows(s + NB + 1);
      if constexpr (MX) {
        decode(0, 0, 0);
        decode(0, 1, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < NM; ++j)
      acc[j >> 1][j & 1] = lin_mfma32<OP>(fp[1][j & 1], fq[1][j >> 1], acc[j >> 1][j & 1]);
  }

  // ---- results ------------------------------------------------------------
  if (KIND == kLinWgrad && slot >= 0) {
    // a partial tile: fp32, [256][256]
    float* o = pl.partials + static_cast<int64_t>(slot) * BQ * kBP;
#pragma unroll
    for (int f = 0; f < FQ; ++f)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int q = 32 * (FQ * wq + f) + (lane & 31);
          const int p = 64 * wp + 32 * k + 8 * r + 4 * half;
          *reinterpret_cast<float4*>(o + q * kBP + p) =
              float4{static_cast<float>(acc[f][k][4 * r]), static_cast<float>(acc[f][k][4 * r + 1]),
                     static_cast<float>(acc[f][k][4 * r + 2]),
                     static_cast<float>(acc[f][k][4 * r + 3])};
        }
    __builtin_amdgcn_s_waitcnt(0);  // loads into LDS of stages past the end
    return;
  }
  float sx[FQ];
  if constexpr (OP == kOpI8) {
#pragma unroll
    for (int f = 0; f < FQ; ++f) {
      int64_t q = q0 + 32 * (FQ * wq + f) + (lane & 31);
      q = q < q_end ? q : q_end - 1;
      sx[f] = g < a.G ? a.sx[lin_row(a, q)] : 0.0f;
    }
  }
  char* out = a.out + (KIND == kLinWgrad ? g * a.o_group : 0) * (a.out_type == kF32 ? 4 : 2);
  lds_handover();  // every wave is done with the last stage's buffer
  // 16-bit results go through LDS (a wave's own part of it) to leave as 128-byte
  // pieces of a row; the chunk swizzle is the operands'
  char* part = lds + wave * (32 * FQ * kRowB);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = p0 + 64 * wp + 32 * k + 8 * r + 4 * half;
      float sw4[4] = {0, 0, 0, 0}, b4[4] = {0, 0, 0, 0};
      if constexpr (OP == kOpI8) {
        const int64_t c = static_cast<int64_t>(gw) * a.np;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t ce = c + (p + e < a.np ? p + e : a.np - 1);
          sw4[e] = a.sw[ce];
          if (a.bias) b4[e] = a.bias[ce];
        }
      }
#pragma unroll
      for (int f = 0; f < FQ; ++f) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = static_cast<float>(acc[f][k][4 * r + e]);
          if constexpr (OP == kOpI8) {
            v[e] = v[e] * sx[f] * sw4[e];
            if (a.bias) v[e] = v[e] + b4[e];
            if (g >= a.G) v[e] = 0.0f;
          }
        }
        const int row = 32 * f + (lane & 31);
        if (a.out_type == kF32) {
          const int64_t q = q0 + 32 * FQ * wq + row;
          if (q < q_end && p < a.np)
            lin_store4(a, out + q * a.ldo * 4, p, v);
        } else {
          uint2 h;
          h.x = lin_round16(v[0], a.out_type) |
                (static_cast<uint32_t>(lin_round16(v[1], a.out_type)) << 16);
          h.y = lin_round16(v[2], a.out_type) |
                (static_cast<uint32_t>(lin_round16(v[3], a.out_type)) << 16);
          *reinterpret_cast<uint2*>(part + row * kRowB + 16 * ((4 * k + r) ^ ((row >> 1) & 7)) +
                                    8 * half) = h;
        }
      }
    }
  if (a.out_type == kF32) return;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 4 * FQ; ++i) {
    const int row = 8 * i + (lane >> 3);
    const int c = (lane & 7) ^ ((row >> 1) & 7);
    const int64_t q = q0 + 32 * FQ * wq + row;
    const int p = p0 + 64 * wp + 8 * c;
    const lin_u32x4_t v = *reinterpret_cast<const lin_u32x4_t*>(part + row * kRowB + 16 * (lane & 7));
    if (q >= q_end) continue;
    uint16_t* o = reinterpret_cast<uint16_t*>(out) + q * a.ldo + p;
    if (a.vec_out == 2 && p + 8 <= a.np) {
      *reinterpret_cast<lin_u32x4_t*>(o) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (p + e < a.np) o[e] = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// ---------------------------------------------------------------------------
// wgrad's units: a group's entries, cut into chunks of at most `cap`, heaviest
// first so that the last tiles to start are the shortest. One workgroup plans.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) lin_plan_kernel(const LinArgs a, const LinPlanArgs pl) {
  __shared__ int32_t size[kLinPlanGroups], parts[kLinPlanGroups];
  for (int g = threadIdx.x; g < a.G; g += 1024) {
    int64_t b = 0, e = a.M;
    if (a.offsets) lin_segment(a, g, &b, &e);
    const int n = e > b ? static_cast<int>(e - b) : 0;
    size[g] = n;
    parts[g] = n > pl.cap ? (n + pl.cap - 1) / pl.cap : 1;
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.G; g += 1024) {
    const int n = size[g], k = parts[g];
    const int len = ((n + k - 1) / k + 63) & ~63;
    int first = 0, slots = 0, splits = 0, units = 0, all_splits = 0;
    for (int o = 0; o < a.G; ++o) {
      const int no = size[o], ko = parts[o];
      const int lo = (no + ko - 1) / ko;
      const int lg = (n + k - 1) / k;
      if (lo > lg || (lo == lg && o < g)) first += ko;
      if (ko > 1) {
        ++all_splits;
        if (o < g) {
          slots += ko;
          ++splits;
        }
      }
      units += ko;
    }
    int64_t b = 0, e = a.M;
    if (a.offsets) lin_segment(a, g, &b, &e);
    for (int i = 0; i < k; ++i) {
      if (first + i >= pl.max_units) break;
      LinUnit u;
      u.g = g;
      const int64_t t0 = static_cast<int64_t>(i) * len, t1 = t0 + len;
      u.t0 = static_cast<int32_t>(b + (t0 < n ? t0 : n));
      u.t1 = static_cast<int32_t>(b + (t1 < n ? t1 : n));
      u.slot = k > 1 && slots + i < pl.max_slots ? slots + i : -1;
      pl.units[first + i] = u;
    }
    if (k > 1 && splits < pl.max_splits) {
      pl.splits[splits].g = g;
      pl.splits[splits].slot0 = slots;
      pl.splits[splits].n = slots + k <= pl.max_slots ? k : 0;
    }
    if (g == 0) {
      pl.counts[0] = units < pl.max_units ? units : pl.max_units;
      pl.counts[1] = all_splits < pl.max_splits ? all_splits : pl.max_splits;
    }
  }
}

// Partial tiles summed in chunk order: grid (tiles * 16, splits), 256 threads,
// 16 rows of a tile each.
__global__ void __launch_bounds__(256) lin_reduce_kernel(const LinArgs a, const LinPlanArgs pl) {
  if (static_cast<int>(blockIdx.y) >= pl.counts[1]) return;
  const LinSplit sp = pl.splits[blockIdx.y];
  const int tiles = pl.npt * pl.nqt;
  const int tile = blockIdx.x >> 4, sub = blockIdx.x & 15;
  const int q0 = tile % pl.nqt * 256 + sub * 16, p0 = tile / pl.nqt * 256;
  const int p = p0 + 4 * (threadIdx.x & 63);
  if (p >= a.np) return;
  const int osize = a.out_type == kF32 ? 4 : 2;
  for (int r = threadIdx.x >> 6; r < 16; r += 4) {
    const int q = q0 + r;
    if (q >= a.nq) return;
    float v[4] = {0, 0, 0, 0};
    for (int i = 0; i < sp.n; ++i) {
      const float* src = pl.partials +
                         (static_cast<int64_t>(sp.slot0 + i) * tiles + tile) * 65536 +
                         (sub * 16 + r) * 256 + (p - p0);
      const float4 f = *reinterpret_cast<const float4*>(src);
      v[0] += f.x;
      v[1] += f.y;
      v[2] += f.z;
      v[3] += f.w;
    }
    lin_store4(a, a.out + (sp.g * a.o_group + q * a.ldo) * osize, p, v);
  }
}

template <int OP, int KIND, int FQ>
int launch(const LinArgs& a, const LinPlanArgs& pl, int64_t grid, hipStream_t s, const char* what) {
  MGQ_REQUIRE(grid < (int64_t(1) << 31), MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  lin_tile_kernel<OP, KIND, FQ><<<static_cast<unsigned>(grid), 512, 0, s>>>(a, pl);
  return check_launch(what);
}

template <int OP, int KIND>
int launch_rows(const LinArgs& a, int fq, hipStream_t s, const char* what) {
  const LinPlanArgs none = {};
  const int64_t grid = lin_row_tiles(a, 64 * fq) * ceil_div(a.np, kBP);
  if (fq == 1) return launch<OP, KIND, 1>(a, none, grid, s, what);
  if (fq == 2) return launch<OP, KIND, 2>(a, none, grid, s, what);
  return launch<OP, KIND, 4>(a, none, grid, s, what);
}

inline bool aligned16(const void* p, int64_t pitch) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (pitch & 15) == 0;
}

}  // namespace

bool lin_tile_takes(const LinArgs& a, int op, int kind) {
  const int es = op == kOpI8 ? 1 : 2;
  if (!aligned16(a.Q, a.ldq) || !aligned16(a.P, a.ldp) || (a.p_group & 15)) return false;
  if (kind == kLinForward) return a.nc * es % 16 == 0;
  if (kind == kLinDgrad) return a.nc % 8 == 0 && a.np % 8 == 0;
  return a.nq % 8 == 0 && a.np % 8 == 0 && a.G <= kLinPlanGroups && a.ldp < (int64_t(1) << 32);
}

int lin_tile_rows(const LinArgs& a, int op, int kind, int fq, hipStream_t s, const char* what) {
  if (kind == kLinDgrad)
    return op == kOpF16 ? launch_rows<kOpF16, kLinDgrad>(a, fq, s, what)
                        : launch_rows<kOpBF16, kLinDgrad>(a, fq, s, what);
  switch (op) {
    case kOpBF16: return launch_rows<kOpBF16, kLinForward>(a, fq, s, what);
    case kOpF16: return launch_rows<kOpF16, kLinForward>(a, fq, s, what);
    case kOpI8: return launch_rows<kOpI8, kLinForward>(a, fq, s, what);
    case kOpMx4: return launch_rows<kOpMx4, kLinForward>(a, fq, s, what);
    default: return launch_rows<kOpMx8, kLinForward>(a, fq, s, what);
  }
}

// Entries per unit at most. With several groups half the average load of a CU
// (entries x tiles / CUs): a heavier group is cut, so that its tiles do not run
// on when the others are done. One group alone is cut so that its tiles fill
// whole rounds of the 256 CUs.
LinPlanSizes lin_plan_sizes(int64_t M, int64_t G, int64_t N, int64_t K) {
  LinPlanSizes z;
  z.tiles = ceil_div(N, 256) * ceil_div(K, kBP);
  int64_t cap = M * z.tiles / 512;
  if (G == 1) {
    double best = 1e300;
    int64_t chunks = 1;
    for (int64_t c = 1; c <= 64 && (c == 1 || M / c >= 256); ++c) {
      // 40 ns an entry of a 256 x 256 tile, 150 ns a partial tile written and read
      const double cost = static_cast<double>(ceil_div(z.tiles * c, 256)) * ceil_div(M, c) * 40e-9 +
                          (c > 1 ? z.tiles * c * 150e-9 : 0.0);
      if (cost < 0.98 * best) {
        best = cost;
        chunks = c;
      }
    }
    cap = ceil_div(M, chunks);
  }
  z.cap = (cap < 1024 && G > 1 ? 1024 : (cap < 64 ? 64 : cap) + 63) & ~int64_t(63);
  const int64_t over = M / z.cap + 1;  // groups longer than cap, and whole chunks
  z.max_splits = M > z.cap ? (over < G ? over : G) : 0;
  z.max_slots = z.max_splits ? over + z.max_splits : 0;
  z.max_units = G + (z.max_splits ? over : 0);
  z.units_off = 256;
  z.splits_off = z.units_off + ceil_div(z.max_units * static_cast<int64_t>(sizeof(LinUnit)), 256) * 256;
  z.partials_off =
      z.splits_off + ceil_div(z.max_splits * static_cast<int64_t>(sizeof(LinSplit)), 256) * 256;
  z.bytes = z.partials_off + z.max_slots * z.tiles * 65536 * 4;
  return z;
}

int lin_tile_wgrad(const LinArgs& a, int op, void* workspace, hipStream_t s, const char* what) {
  const LinPlanSizes z = lin_plan_sizes(a.M, a.G, a.nq, a.np);
  char* ws = static_cast<char*>(workspace);
  LinPlanArgs pl = {};
  pl.counts = reinterpret_cast<int32_t*>(ws);
  pl.units = reinterpret_cast<LinUnit*>(ws + z.units_off);
  pl.splits = reinterpret_cast<LinSplit*>(ws + z.splits_off);
  pl.partials = reinterpret_cast<float*>(ws + z.partials_off);
  pl.npt = static_cast<int>(ceil_div(a.np, kBP));
  pl.nqt = static_cast<int>(ceil_div(a.nq, 256));
  pl.cap = static_cast<int>(z.cap);
  pl.max_units = static_cast<int>(z.max_units);
  pl.max_splits = static_cast<int>(z.max_splits);
  pl.max_slots = static_cast<int>(z.max_slots);
  pl.deal = a.G >= 64;
  lin_plan_kernel<<<1, 1024, 0, s>>>(a, pl);
  if (int rc = check_launch(what)) return rc;
  const int64_t grid = (pl.deal ? ceil_div(z.max_units, 8) * 8 : z.max_units) * z.tiles;
  const int rc = op == kOpF16 ? launch<kOpF16, kLinWgrad, 4>(a, pl, grid, s, what)
                              : launch<kOpBF16, kLinWgrad, 4>(a, pl, grid, s, what);
  if (rc || z.max_splits == 0) return rc;
  const dim3 rg(static_cast<unsigned>(z.tiles * 16), static_cast<unsigned>(z.max_splits));
  lin_reduce_kernel<<<rg, 256, 0, s>>>(a, pl);
  return check_launch(what);
}

}  // namespace mgq
