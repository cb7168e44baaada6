// Large tiles of the matrix products (linear_common.h has the products and their
// operands).
//
// Tile kernel: 512 threads = 8 waves, 2 along q and 4 along p, one workgroup
// per CU. A wave owns 32 FQ x 32 FP outputs as blocks of a 32x32 MFMA (FQ = 4,
// FP = 2: a 256 x 256 tile, 128 fp32 accumulators per lane).
//
//   - A stage is 128 bytes of every row: 64 16-bit or 128 int8 elements of the
//     contraction, four K-steps of one MFMA depth each. Rows that start and end on
//     16-byte boundaries go from memory straight into LDS
//     (global_load_lds_dwordx4, 16 bytes a lane), two to four stages deep. Other rows
//     (STAGED) go through registers, loaded a stage ahead of their way into LDS,
//     with 16-byte loads at any address; a piece that a row ends in is masked, and
//     read element by element only where the 16 bytes would leave the tensor.
//     What lies past the contraction's end is zeros; rows past the operand's end
//     repeat its last row and their results are not stored.
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
//     LDS reads and of the loads of the stage that takes the buffer released by
//     the last barrier. The last K-step of a stage runs after the barrier, over the
//     first reads of the next stage.
//
// Measured (MI355X; the library's bf16 product of 8192^3 reaches 1390 to 1650 TFLOP/s on
// the same cards, MFMA busy 85 to 88 %, its int8 one 2120 to 2460 TOP/s):
//   524288 gathered rows x 128 experts [1536, 2048] bf16: 2.93 ms, 1130 TFLOP/s,
//     MFMA busy 67 % at a clock of 1.56 GHz;
//   131072 rows x the same experts as MXFP4 codes: 0.77 ms, 1070 TFLOP/s (64 % busy);
//   8191 rows x int8 [14336, 4096]: 0.44 ms, 2200 TOP/s (61 % busy);
//   dgrad and wgrad of 131072 rows x 128 experts [2048, 768] bf16: 0.90 to 0.94 ms,
//     880 to 910 TFLOP/s (60 and 48 % busy).
// Long contractions are bound by the stage: with every CU loading, its 64 KiB take
// 1.5 to 1.75 us to come where the MFMAs need 1.1. Short ones are bound by the first
// loads (3 us under load) and the results. Two stages of 64-byte rows, four waves of
// 128 x 128, one K-step more between loads and use, and wave priorities measured no
// faster.
#include "linear_tile.h"

namespace mgq {
namespace {

constexpr int kLdsMax = 160 * 1024;
constexpr int kCUs = 256;
constexpr int kSteps = 4;    // K-steps per stage
constexpr int kRowB = 128;   // bytes of a plain row per stage

__device__ uint32_t g_lin_zeros[64];  // never written: what lies past an operand's end

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) lin_u32x4_t lds_u32x4;
typedef short lin_s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) lin_s16x4_t lds_s16x4;
typedef const __attribute__((address_space(4))) int32_t* const_i32_ptr;

// Wait until at most VM of this wave's loads are in flight (VM < 0: whatever is)
// and its LDS accesses are done, then for the other waves. The memory clobber
// orders the LDS accesses for the compiler as __syncthreads would, without its
// wait for every load.
template <int VM>
__device__ __forceinline__ void stage_barrier() {
  static_assert(VM <= 63, "vmcnt range");
  if constexpr (VM >= 0)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
  else
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 16 bytes (4; 1, widened to a dword) per lane from `src` to LDS at
// dst + 16 (4; 4) * lane. (One wait state between the write of m0 and its use.)
__device__ __forceinline__ void dma16(uint32_t dst, uint64_t src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src)
               : "memory");
}
__device__ __forceinline__ void dma4(uint32_t dst, uint64_t src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(src)
               : "memory");
}
__device__ __forceinline__ void dma1(uint32_t dst, uint64_t src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off" ::"s"(dst), "v"(src)
               : "memory");
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

__device__ __forceinline__ lin_u32x4_t load16(uint64_t src) {
  const lin_u128_u_t u = *reinterpret_cast<const lin_u128_u_t*>(src);
  return lin_u32x4_t{u.v[0], u.v[1], u.v[2], u.v[3]};
}
// The first n bytes at `src` (n <= 0: none, n >= 16: all), zeros after them. 16
// bytes are read where they lie before `end`, single elements otherwise.
template <int ES>
__device__ __forceinline__ lin_u32x4_t load_cut(uint64_t src, int n, uint64_t end) {
  lin_u32x4_t r = {0, 0, 0, 0};
  if (n <= 0) return r;
  if (src + 16 <= end) {
    r = load16(src);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int left = n - 4 * i;
      r[i] &= left >= 4 ? 0xffffffffu : left > 0 ? (1u << (8 * left)) - 1u : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i)
      if (i * ES < n) {
        const uint32_t v = ES == 2 ? *reinterpret_cast<const uint16_t*>(src + 2 * i)
                                   : *reinterpret_cast<const uint8_t*>(src + i);
        r[i * ES / 4] |= v << (8 * ((i * ES) & 3));
      }
  }
  return r;
}

// The low cut >> 8 bytes shifted out, then all but the low (cut & 255) cleared.
__device__ __forceinline__ lin_u32x4_t cut16(lin_u32x4_t v, int cut) {
  const int d = cut >> 8, m = cut & 255;
  if (__any(d != 0)) {
    // whole dwords, then bytes
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      const bool go = (d >> 2) > w;
      v = lin_u32x4_t{go ? v[1] : v[0], go ? v[2] : v[1], go ? v[3] : v[2], go ? 0u : v[3]};
    }
    const uint32_t s = 8 * (d & 3);
    v = lin_u32x4_t{__builtin_amdgcn_alignbit(v[1], v[0], s), __builtin_amdgcn_alignbit(v[2], v[1], s),
                    __builtin_amdgcn_alignbit(v[3], v[2], s), v[3] >> s};
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = m - 4 * i;
    v[i] &= left >= 4 ? 0xffffffffu : left > 0 ? (1u << (8 * left)) - 1u : 0u;
  }
  return v;
}

template <int OP>
constexpr int mx_stage_bytes(int bp) {
  return OP == kOpMx4 ? bp * 32 + bp * 8 : bp * 64 + bp * 8;
}

template <int OP, int KIND, int FQ, int FP, bool STAGED>
__global__ void __launch_bounds__(512, 1) lin_tile_kernel(const LinArgs a, const LinPlanArgs pl) {
  constexpr bool PT = KIND != kLinForward;
  constexpr bool WGRAD = KIND == kLinWgrad || KIND == kLinWgradGather;
  constexpr bool GATHER = KIND == kLinWgradGather;
  constexpr bool QT = WGRAD;
  constexpr bool MX = lin_is_mx<OP>();
  constexpr int ES = lin_esize<OP>();
  constexpr int BQ = 64 * FQ, BP = 128 * FP;
  constexpr int QB = BQ * kRowB;                 // Q bytes per stage
  constexpr int PB = MX ? mx_stage_bytes<OP>(BP) : BP * kRowB;  // and P bytes
  // buffers of stages: where two whole ones leave room, Q has a third, so that only
  // P's loads have to come within the period they are issued in
  constexpr int NBP = STAGED ? 2 : kLdsMax / (QB + PB) < 4 ? kLdsMax / (QB + PB) : 4;
  constexpr bool RING = GATHER && !STAGED;       // the gathered rows' indexes come through LDS
  constexpr int NBQ = !STAGED && !RING && NBP == 2 && 3 * QB + 2 * PB <= kLdsMax ? 3 : NBP;
  constexpr int RING_AT = NBQ * QB + NBP * PB;
  constexpr int LDS = RING_AT + (RING ? 8 * 512 : 0);
  constexpr int EPI = BQ * BP * 2;               // 16-bit results on their way out
  constexpr int VQ = FQ;                         // 16-byte loads per lane and stage: Q,
  constexpr int per = OP == kOpMx4 ? 2 : 4;      // (MX: 16-byte pieces of a row's codes)
  constexpr int VC = OP == kOpMx8 ? FP : 1;      // codes, and one of a scale byte,
  constexpr int VP = MX ? VC + 1 : 2 * FP;       // or a dense P
  constexpr int V = VQ + VP;
  constexpr int NM = FP * FQ;                    // MFMAs per K-step
  constexpr int EK = kRowB / ES;                 // contraction elements per stage
  static_assert(NBP >= 2 && (NBP - 2) * V <= 63, "stages");
  static_assert(!QT || FQ >= 2, "transposed Q tiles are 128 or 256 wide");
  __shared__ __attribute__((aligned(1024))) char lds[LDS > EPI ? LDS : EPI];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wq = wave >> 2, wp = wave & 3;
  const int half = lane >> 5;

  // ---- which tile -------------------------------------------------------
  // wgrad: the host's bound on the work list is loose (it does not know the groups'
  // lengths), so that a workgroup takes every gridDim.x'th item instead of leaving
  // the holes to workgroups of their own. The products over rows have few holes,
  // and one tile a workgroup: taking several, with the next one's first loads before
  // the results of the last, measured 2 to 4 % slower in long contractions.
  for (uint32_t item = blockIdx.x;; item += gridDim.x) {
    int g, p0, slot = -1;
    int q0, q_end;                 // rows of Q (forward, dgrad) or of the output (wgrad)
    int c_begin = 0, c_len = a.nc;  // contraction range
    if constexpr (WGRAD) {
      LinUnit u;
      int tile;
      const int found = lin_find_unit(a, pl, item, &u, &tile);
      if (found == 0) return;
      if (found < 0) continue;
      g = u.g;
      slot = u.slot;
      c_begin = u.t0;
      c_len = u.t1 - u.t0;
      q0 = tile % pl.nqt * BQ;
      p0 = tile / pl.nqt * BP;
      q_end = a.nq;
    } else {
      LinTile t;
      if (!lin_find_tile<BQ>(a, (a.np + BP - 1) / BP, &t)) return;
      g = t.g;
      p0 = t.pt * BP;
      q0 = t.q0;
      q_end = t.q_end;
      if (g >= a.G) c_len = 0;  // entries of no group: zeros
    }
    const int gw = WGRAD || g >= a.G ? 0 : g;
    const char* Pg = a.P + gw * a.p_group;
    const int n_stages = (c_len + EK - 1) / EK;

    // ---- loads ------------------------------------------------------------
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char*)lds));
    const uint64_t zeros = reinterpret_cast<uint64_t>(g_lin_zeros);
    // plain rows: load i of a wave takes rows 8 (n wave + i) .. + 7, lane l the place
    // l % 8 of row l / 8, which holds the row's chunk ^ its swizzle (that depends on
    // i's parity only)
    const int ch0 = (lane & 7) ^ ((lane >> 4) & 7), ch1 = ch0 ^ 4;
    // transposed rows, W columns: a load takes 512 / W of the stage's 64 contraction
    // rows, a wave eight of them; lane l the place l % (W / 8) of its row, which holds
    // the row's chunk ^ 4 (row % 4)
    auto tr_row = [&](int W, int i) { return 8 * wave + (512 / W) * i + lane / (W / 8); };
    auto tr_col = [&](int W, int i) { return 8 * ((lane % (W / 8)) ^ (4 * (tr_row(W, i) & 3))); };
    // MX: mxfp4 codes and the scales of 128 rows are four loads, which waves 4..7
    // repeat so that every wave has the same loads to wait for
    const int mx_wave = FP == 2 ? wave : wave & 3;
    uint64_t qp[VQ], pp[VP];
    if constexpr (QT) {
#pragma unroll
      for (int i = 0; i < VQ; ++i) {
        int col = q0 + tr_col(BQ, i);
        if (!STAGED) col = col + 8 <= a.nq ? col : a.nq - 8;
        if (STAGED) col = col < a.nq ? col : a.nq - 1;
        qp[i] = reinterpret_cast<uint64_t>(a.Q) + (c_begin + tr_row(BQ, i)) * a.ldq + 2 * static_cast<int64_t>(col);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VQ; ++i) {
        int q = q0 + 8 * (VQ * wave + i) + (lane >> 3);
        q = q < q_end ? q : q_end - 1;
        const int64_t row = KIND == kLinForward ? lin_row(a, q) : q;
        qp[i] = reinterpret_cast<uint64_t>(a.Q) + row * a.ldq + 16 * (((VQ * wave + i) & 1) ? ch1 : ch0);
      }
    }
    if constexpr (MX) {
      const uint8_t* Psg = a.Ps + static_cast<int64_t>(gw) * a.np * (a.nc / 32);
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const int r = (64 / per) * (VC * (per == 2 ? mx_wave : wave) + i) + lane / per;
        const int pos = lane % per;
        const int c = per == 2 ? pos ^ ((r >> 3) & 1) : pos ^ ((r >> 2) & 3);
        const int p = p0 + r < a.np ? p0 + r : a.np - 1;
        pp[i] = reinterpret_cast<uint64_t>(Pg) + p * a.ldp + 16 * c;
      }
      const int r = 32 * mx_wave + (lane >> 1);
      const int p = p0 + r < a.np ? p0 + r : a.np - 1;
      pp[VC] = reinterpret_cast<uint64_t>(Psg) + static_cast<int64_t>(p) * (a.nc / 32) + (lane & 1);
    } else if constexpr (PT) {
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        int col = p0 + tr_col(BP, i);
        if (!STAGED) col = col + 8 <= a.np ? col : a.np - 8;
        if (STAGED) col = col < a.np ? col : a.np - 1;
        // (gathered: the row is added when it is known)
        pp[i] = reinterpret_cast<uint64_t>(Pg) + 2 * static_cast<int64_t>(col) +
                (GATHER ? 0 : (c_begin + tr_row(BP, i)) * a.ldp);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        const int r = 8 * (VP * wave + i) + (lane >> 3);
        const int p = p0 + r < a.np ? p0 + r : a.np - 1;
        pp[i] = reinterpret_cast<uint64_t>(Pg) + p * a.ldp + 16 * (i & 1 ? ch1 : ch0);
      }
    }
    // STAGED: where the operands end
    uint64_t q_stop = 0, p_stop = 0;
    if constexpr (STAGED) {
      const int64_t q_rows = KIND == kLinForward ? a.n_rows : a.M;
      const int64_t q_cols = QT ? a.nq : a.nc;
      q_stop = reinterpret_cast<uint64_t>(a.Q) + (q_rows - 1) * a.ldq + q_cols * ES;
      const int64_t p_rows = WGRAD ? a.n_rows : KIND == kLinDgrad ? a.nc : a.np;
      const int64_t p_cols = PT ? a.np : a.nc;
      p_stop = reinterpret_cast<uint64_t>(Pg) + (p_rows - 1) * a.ldp + p_cols * ES;
    }

    // gathered wgrad: the rows of X that this wave loads in the next stage, 8 a stage.
    // RING: their indexes come into LDS 64 at a time (8 stages), at least six stages
    // before their use, into the wave's ring of two such blocks, and from there a stage
    // ahead: a load into registers would be waited for with every load into LDS issued
    // before it, and scalar loads return out of order with the LDS reads, which then
    // wait for all of them (2.6 us a stage against 1.5).
    int rows[8], rows_next[8];
    const uint32_t ring = lds0 + RING_AT + wave * 512;
    auto ring_fetch = [&](int block) {
      if constexpr (RING) {
        const int t0 = c_begin + (8 * block + (lane >> 3)) * EK + 8 * wave + (lane & 7);
        const int last = c_begin + c_len - 1;
        dma4(ring + (block & 1) * 256,
             reinterpret_cast<uint64_t>(a.row_index) + 4 * static_cast<int64_t>(t0 < last ? t0 : last));
      }
    };
    auto load_rows = [&](int st) {
      if constexpr (RING) {
        rows_next[0] = *reinterpret_cast<const __attribute__((address_space(3))) int32_t*>(
            ring + ((st >> 3) & 1) * 256 + ((st & 7) * 8 + (lane & 7)) * 4);
      } else if constexpr (GATHER) {
        const int t0 = c_begin + st * EK + 8 * wave;  // (below 2^31: see the entry points)
        const int last = c_begin + c_len - 1;
        const const_i32_ptr index =
            reinterpret_cast<const_i32_ptr>(reinterpret_cast<uint64_t>(a.row_index));
#pragma unroll
        for (int i = 0; i < 8; ++i) rows_next[i] = index[t0 + i < last ? t0 + i : last];
      }
    };
    auto take_rows = [&]() {  // (clamped here, so that no load is waited for above)
      if constexpr (GATHER) {
        // (X may have more rows than an index can name)
        const int top = a.n_rows < 0x7fffffff ? static_cast<int>(a.n_rows) - 1 : 0x7fffffff;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int v = RING ? __builtin_amdgcn_readlane(rows_next[0], i) : rows_next[i];
          const int r = v < 0 ? 0 : v;
          rows[i] = r < top ? r : top;
        }
      }
    };

    // load i of stage st: where it comes from (advancing the pointer), how many bytes
    // of it exist, and its place in the stage
    auto source = [&](int i, int st, uint64_t* src, int* n, uint32_t* dst) __attribute__((
                      always_inline)) {
      const int left = c_len - st * EK;  // contraction elements
      if (i < VQ) {
        *dst = (VQ * wave + i) * 1024;
        *src = qp[i];
        if constexpr (QT) {
          *n = tr_row(BQ, i) < left ? 16 : 0;
          qp[i] += EK * a.ldq;
        } else {
          *n = left * ES - 16 * (((VQ * wave + i) & 1) ? ch1 : ch0);
          qp[i] += kRowB;
        }
        return;
      }
      const int k = i - VQ;
      *src = pp[k];
      if constexpr (MX) {
        if (k < VC) {
          const int at = VC * (per == 2 ? mx_wave : wave) + k;
          const int r = (64 / per) * at + lane / per;
          const int pos = lane % per;
          const int c = per == 2 ? pos ^ ((r >> 3) & 1) : pos ^ ((r >> 2) & 3);
          *dst = at * 1024;
          *n = 32 * (c * 2 / per) < left ? 16 : 0;  // whole MX groups
          pp[k] += 16 * per;
        } else {
          *dst = BP * 16 * per + mx_wave * 256;
          *n = 32 * (lane & 1) < left ? 1 : 0;
          pp[k] += 2;
        }
      } else if constexpr (PT) {
        *dst = (VP * wave + k) * 1024;
        *n = tr_row(BP, k) < left ? 16 : 0;
        if constexpr (GATHER) {
          constexpr int RP = 512 / BP;  // rows per load
          int64_t at = rows[RP * k] * a.ldp;
#pragma unroll
          for (int j = 1; j < RP; ++j) at = lane / (BP / 8) == j ? rows[RP * k + j] * a.ldp : at;
          *src += at;
        } else {
          pp[k] += EK * a.ldp;
        }
      } else {
        *dst = (VP * wave + k) * 1024;
        *n = left * ES - 16 * (k & 1 ? ch1 : ch0);
        pp[k] += kRowB;
      }
    };
    auto is_scale = [&](int i) { return MX && i == V - 1; };
    // straight into LDS (rows are whole pieces: n is 16 or more, or nothing is left)
    auto load = [&](int i, int st, uint32_t buf) __attribute__((always_inline)) {
      uint64_t src;
      int n;
      uint32_t dst;
      source(i, st, &src, &n, &dst);
      if (is_scale(i))
        dma1(buf + dst, n > 0 ? src : zeros);
      else
        dma16(buf + dst, n > 0 ? src : zeros);
    };
    // through registers
    lin_u32x4_t hold[STAGED ? V : 1];
    int cut[STAGED ? V : 1];  // bytes kept | bytes shifted out << 8
    const bool tiny = STAGED && (q_stop - reinterpret_cast<uint64_t>(a.Q) < 16 ||
                                 p_stop - reinterpret_cast<uint64_t>(Pg) < 16);
    auto fetch = [&](int i, int st) __attribute__((always_inline)) {
      uint64_t src;
      int n;
      uint32_t dst;
      source(i, st, &src, &n, &dst);
      const bool tr = i < VQ ? QT : PT;
      if (is_scale(i)) {
        const uint32_t v = *reinterpret_cast<const uint8_t*>(n > 0 ? src : zeros);
        hold[i] = lin_u32x4_t{v, 0, 0, 0};
      } else if (tr || (MX && i >= VQ)) {
        // a transposed row may end inside the piece: the columns past its end are not
        // stored, but nothing is read past the tensor's end
        const uint64_t stop = i < VQ ? q_stop : p_stop;
        if (n > 0 && src + 16 > stop)
          hold[i] = load_cut<ES>(src, static_cast<int>(stop - src), stop);
        else
          hold[i] = load16(n > 0 ? src : zeros);
      } else if ((st + 1) * EK <= c_len) {
        hold[i] = load16(src);
      } else {
        // the stage in which the rows end: n of the 16 bytes exist. They are loaded
        // whole (from 16 bytes before the operand's end if they would pass it) and cut on
        // the way into LDS, so that no load is waited for here.
        const uint64_t stop = i < VQ ? q_stop : p_stop;
        const int m = n < 0 ? 0 : n > 16 ? 16 : n;
        if (tiny) {
          hold[i] = load_cut<ES>(src, m, stop);
          cut[i] = 16;
        } else {
          const bool past = m > 0 && src + 16 > stop;
          hold[i] = load16(m == 0 ? zeros : past ? stop - 16 : src);
          cut[i] = m | (past ? static_cast<int>(src + 16 - stop) << 8 : 0);
        }
      }
    };
    auto put = [&](int i, int st, uint32_t buf) __attribute__((always_inline)) {
      const int k = i - VQ;
      const bool plain = i < VQ ? !QT : !PT && !MX;
      if (plain && (st + 1) * EK > c_len) hold[i] = cut16(hold[i], cut[i]);
      uint32_t dst;
      if (i < VQ) dst = (VQ * wave + i) * 1024;
      else if (is_scale(i)) dst = BP * 16 * per + mx_wave * 256;
      else if (MX) dst = (VC * (per == 2 ? mx_wave : wave) + k) * 1024;
      else dst = (VP * wave + k) * 1024;
      if (is_scale(i))
        *reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(buf + dst + 4 * lane) = hold[i][0];
      else
        *reinterpret_cast<lds_u32x4*>(buf + dst + 16 * lane) = hold[i];
    };

    // ---- LDS reads of a K-step's operands -----------------------------------
    // plain: chunk 2 ks + half of the row (MX: 4 half + ks, so that a half-wave
    // keeps to its MX group)
    const int sw = (lane >> 1) & 7;
    uint32_t qa[4], pa[4];  // plain: by K-step; transposed: by block
    const int j4 = (lane >> 2) & 3;
    const uint32_t tr_lane = ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t c = 16 * ((MX ? 4 * half + k : 2 * k + half) ^ sw);
      qa[k] = QT ? (8 * half + j4) * (2 * BQ) + (((FQ * wq + k) ^ j4) * 64) + tr_lane
                 : (32 * FQ * wq + (lane & 31)) * kRowB + c;
      pa[k] = PT ? (8 * half + j4) * (2 * BP) + (((FP * wp + (k & (FP - 1))) ^ j4) * 64) + tr_lane
                 : (32 * FP * wp + (lane & 31)) * kRowB + c;
    }
    uint32_t code_at[2], scale_at = 0;
    if constexpr (MX) {
      const int r = 32 * FP * wp + (lane & 31);
#pragma unroll
      for (int k = 0; k < per / 2; ++k) {
        const int c = per == 2 ? half : 2 * half + k;
        const int pos = per == 2 ? c ^ ((r >> 3) & 1) : c ^ ((r >> 2) & 3);
        code_at[k] = r * 16 * per + 16 * pos;
      }
      scale_at = BP * 16 * per + (2 * r + half) * 4;
    }
    lin_u32x4_t fq[2][FQ], fp[2][FP];
    lin_u32x4_t codes[FP][2];
    uint32_t scale[FP];
    auto read_q = [&](int b, int f, int ks, uint32_t buf) {
      if constexpr (QT)
        fq[b][f] = read_tr(buf + qa[f] + 16 * ks * (2 * BQ), 2 * BQ);
      else
        fq[b][f] = read16(buf + qa[ks] + f * 32 * kRowB);
    };
    auto read_p = [&](int b, int f, int ks, uint32_t buf) {
      if constexpr (PT)
        fp[b][f] = read_tr(buf + pa[f] + 16 * ks * (2 * BP), 2 * BP);
      else
        fp[b][f] = read16(buf + pa[ks] + f * 32 * kRowB);
    };
    auto read_codes = [&](int f, uint32_t buf) {
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
    // read r of a K-step (dense: p0 q0 p1 .. q1 ..; MX: the q only)
    constexpr int NR = MX ? FQ : FQ + FP;
    auto read = [&](int r, int b, int ks, uint32_t qbuf, uint32_t pbuf) {
      if constexpr (MX) {
        read_q(b, r, ks, qbuf);
      } else {
        if (r == 0) read_p(b, 0, ks, pbuf);
        else if (r == 1) read_q(b, 0, ks, qbuf);
        else if (r <= FP) read_p(b, r - 1, ks, pbuf);
        else read_q(b, r - FP, ks, qbuf);
      }
    };

    typedef typename LinAcc<OP>::t32 acc_t;
    acc_t acc[FQ][FP];
#pragma unroll
    for (int i = 0; i < FQ; ++i)
#pragma unroll
      for (int j = 0; j < FP; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    auto mfma = [&](int b, int j) {
      acc[j / FP][j % FP] = lin_mfma32<OP>(fp[b][j % FP], fq[b][j / FP], acc[j / FP][j % FP]);
    };
    auto decode_all = [&](int b, int ks) {
#pragma unroll
      for (int f = 0; f < FP; ++f) decode(b, f, ks);
    };

    // Slot t of a stage's period (four K-steps of NM MFMAs; the first K-step's MFMAs
    // are the previous stage's last): the reads of the next K-step come first, so
    // that none is young at the barrier. The loads into the buffers that the barrier
    // released (P of stage s + NBP - 1, then Q of stage s + NBQ - 1) are spread over
    // the period, because a load instruction occupies the address unit of the CU for
    // 16 cycles and all eight waves issue theirs in the same slots; with two buffers
    // over its first half, because the next barrier waits for them. STAGED: what was
    // loaded in the last period goes into LDS, and the next stage's loads take its
    // registers.
    constexpr int SPREAD = NBP == 2 ? kSteps / 2 : kSteps;
    constexpr int RPS = (NR + NM - 1) / NM;
    constexpr int WAIT = STAGED ? -1 : (NBQ - 2) * VQ + (NBP - 2) * VP;
    auto q_at = [&](int i) { return lds0 + i * QB; };
    auto p_at = [&](int i) { return lds0 + NBQ * QB + i * PB; };
    auto slot_reads = [&](int j, int b, int ks, uint32_t qbuf, uint32_t pbuf) __attribute__((
                          always_inline)) {
#pragma unroll
      for (int r = j * RPS; r < (j + 1) * RPS && r < NR; ++r) read(r, b, ks, qbuf, pbuf);
    };
    auto slot_loads = [&](int t, int s, uint32_t qbuf, uint32_t pbuf) __attribute__((always_inline)) {
#pragma unroll
      for (int k = t * V / (NM * SPREAD); k < (t + 1) * V / (NM * SPREAD) && k < V; ++k) {
        const int i = k < VP ? VQ + k : k - VP;
        const uint32_t buf = k < VP ? pbuf : qbuf;
        const int st = s + (k < VP ? NBP : NBQ) - 1;
        if constexpr (STAGED) {
          put(i, st, buf);
          fetch(i, st + 1);
        } else {
          load(i, st, buf);
        }
      }
    };
    if (n_stages > 0) {
      if constexpr (STAGED) {
        load_rows(0);
        take_rows();
#pragma unroll
        for (int i = 0; i < V; ++i) fetch(i, 0);
        load_rows(1);
        take_rows();
#pragma unroll
        for (int i = 0; i < V; ++i) {
          put(i, 0, i < VQ ? q_at(0) : p_at(0));
          fetch(i, 1);
        }
        load_rows(2);
      } else {
        if constexpr (RING) {
          ring_fetch(0);
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int st = 0; st < NBQ - 1; ++st) {
          if (st < NBP - 1) {
            load_rows(st);
            take_rows();
#pragma unroll
            for (int i = VQ; i < V; ++i) load(i, st, p_at(st));
          }
#pragma unroll
          for (int i = 0; i < VQ; ++i) load(i, st, q_at(st));
        }
        load_rows(NBP - 1);
      }
      stage_barrier<WAIT>();
      take_rows();
      if constexpr (MX) {
#pragma unroll
        for (int f = 0; f < FP; ++f) read_codes(f, p_at(0));
      }
      uint32_t wqb = q_at(NBQ - 1), wpb = p_at(NBP - 1);
#pragma unroll
      for (int r = 0; r < NR; ++r) read(r, 0, 0, q_at(0), p_at(0));
#pragma unroll
      for (int j = 0; j < NM; ++j) slot_loads(j, 0, wqb, wpb);
      if constexpr (MX) decode_all(0, 0);
      __builtin_amdgcn_sched_barrier(0);
      int rq = 0, rp = 0;
      for (int s = 0; s < n_stages; ++s) {
        const uint32_t qbuf = q_at(rq), pbuf = p_at(rp);
        if (RING && (s & 7) == 0) ring_fetch((s >> 3) + 1);
        load_rows(s + NBP + (STAGED ? 1 : 0));
#pragma unroll
        for (int ks = 1; ks < kSteps; ++ks) {
          const int b = (ks - 1) & 1;
#pragma unroll
          for (int j = 0; j < NM; ++j) {
            mfma(b, j);
            slot_reads(j, b ^ 1, ks, qbuf, pbuf);
            slot_loads(ks * NM + j, s, wqb, wpb);
            if constexpr (MX) {
              if (j % FQ == 0) decode(b ^ 1, j / FQ, ks);
            }
            if (j & 1) __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (s + 1 == n_stages) break;
        rq = rq + 1 == NBQ ? 0 : rq + 1;
        rp = rp + 1 == NBP ? 0 : rp + 1;
        const uint32_t next_q = q_at(rq), next_p = p_at(rp);
        wqb = qbuf;
        wpb = pbuf;
        stage_barrier<WAIT>();
        take_rows();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MX) {
#pragma unroll
          for (int f = 0; f < FP; ++f) read_codes(f, next_p);
        }
#pragma unroll
        for (int j = 0; j < NM; ++j) {
          mfma(1, j);
          slot_reads(j, 0, 0, next_q, next_p);
          slot_loads(j, s + 1, wqb, wpb);
          if (j & 1) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (MX) decode_all(0, 0);
      }
#pragma unroll
      for (int j = 0; j < NM; ++j) mfma(1, j);
    }

    // ---- results ------------------------------------------------------------
    float sx[FQ];
    if constexpr (OP == kOpI8) {
#pragma unroll
      for (int f = 0; f < FQ; ++f) {
        int q = q0 + 32 * (FQ * wq + f) + (lane & 31);
        q = q < q_end ? q : q_end - 1;
        sx[f] = g < a.G ? a.sx[lin_row(a, q)] : 0.0f;
      }
    }
    char* out = a.out + (WGRAD ? g * a.o_group : 0) * (a.out_type == kF32 ? 4 : 2);
    int64_t ldo = a.ldo;
    const bool partial = WGRAD && slot >= 0;
    if (partial) {  // fp32, [BQ][BP]
      ldo = BP;
      out = reinterpret_cast<char*>(pl.partials + static_cast<int64_t>(slot) * BQ * BP -
                                    static_cast<int64_t>(q0) * BP - p0);
    }
    lds_handover();  // every wave is done with the last stage's buffer
    // Results go through LDS (a wave's own part of it) to leave as whole pieces of a
    // row: 64 columns of 16-bit results or 32 of fp32 at a time, rows of 128 bytes
    // (64 at FP = 1) with the operands' chunk swizzle.
    auto store_out = [&](auto type) __attribute__((always_inline)) {
      constexpr int T = decltype(type)::value;
      constexpr int OS = T == kF32 ? 4 : 2;
      constexpr int KP = T == kF32 || FP == 1 ? 1 : 2;  // 32-column blocks per pass
      constexpr int RB = 32 * KP * OS, CH = RB / 16;    // bytes and 16-byte chunks of a row
      constexpr int EC = 16 / OS;                       // results per chunk
      auto swizzle = [](int row) { return CH == 8 ? (row >> 1) & 7 : (row >> 2) & 3; };
      char* part = lds + wave * (32 * FQ * RB);
#pragma unroll
      for (int k0 = 0; k0 < FP; k0 += KP) {
#pragma unroll
        for (int k = k0; k < k0 + KP; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int p = p0 + 32 * (FP * wp + k) + 8 * r + 4 * half;
            float sw4[4] = {0, 0, 0, 0}, b4[4] = {0, 0, 0, 0};
            if constexpr (OP == kOpI8) {
              const int64_t c = static_cast<int64_t>(gw) * a.np;
              lin_load4(a.sw + c, p, a.np, sw4);
              if (a.bias) lin_load4(a.bias + c, p, a.np, b4);
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
              if constexpr (T == kF32) {
                *reinterpret_cast<float4*>(part + row * RB + 16 * ((2 * r + half) ^ swizzle(row))) =
                    float4{v[0], v[1], v[2], v[3]};
              } else {
                uint2 h;
                h.x = lin_pack2<T>(v[0], v[1]);
                h.y = lin_pack2<T>(v[2], v[3]);
                *reinterpret_cast<uint2*>(part + row * RB +
                                          16 * ((4 * (k - k0) + r) ^ swizzle(row)) + 8 * half) = h;
              }
            }
          }
        __builtin_amdgcn_wave_barrier();
        // the loop stays small: it is most of what a short contraction runs
#pragma unroll 4
        for (int i = 0; i < 32 * FQ * CH / 64; ++i) {
          const int row = (64 / CH) * i + lane / CH;
          const int c = (lane % CH) ^ swizzle(row);
          const int q = q0 + 32 * FQ * wq + row;
          const int p = p0 + 32 * (FP * wp + k0) + EC * c;
          const lin_u32x4_t v =
              *reinterpret_cast<const lin_u32x4_t*>(part + row * RB + 16 * (lane % CH));
          if (q >= q_end) continue;
          char* o = out + (static_cast<int64_t>(q) * ldo + p) * OS;
          if (p + EC <= a.np) {  // (at any address)
            lin_u128_u_t u;
#pragma unroll
            for (int e = 0; e < 4; ++e) u.v[e] = v[e];
            *reinterpret_cast<lin_u128_u_t*>(o) = u;
          } else {
            for (int e = 0; e < EC && p + e < a.np; ++e) {
              if constexpr (T == kF32)
                reinterpret_cast<uint32_t*>(o)[e] = e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3];
              else
                reinterpret_cast<uint16_t*>(o)[e] = static_cast<uint16_t>(
                    (e < 2 ? v[0] : e < 4 ? v[1] : e < 6 ? v[2] : v[3]) >> (16 * (e & 1)));
            }
          }
        }
        if (k0 + KP < FP) __builtin_amdgcn_wave_barrier();
      }
    };
    if (a.out_type == kF32 || partial) {
      if constexpr (OP == kOpI8 || KIND != kLinForward) store_out(std::integral_constant<int, kF32>{});
    } else if (a.out_type == kF16) {
      if constexpr (OP == kOpI8 || OP == kOpF16) store_out(std::integral_constant<int, kF16>{});
    } else {
      if constexpr (OP != kOpF16) store_out(std::integral_constant<int, kBF16>{});
    }
    if constexpr (!WGRAD) return;
    stage_barrier<-1>();  // every wave has its results out of LDS (they need not be stored yet)
  }
}

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

template <int OP, int KIND, int FQ, int FP, bool STAGED>
int launch(const LinArgs& a, const LinPlanArgs& pl, int64_t grid, hipStream_t s, const char* what) {
  const int64_t most = KIND == kLinWgrad || KIND == kLinWgradGather ? 2 * kCUs : grid;
  MGQ_REQUIRE(most < kLinTileGrid && grid < (int64_t(1) << 31), MGQ_ERR_SHAPE,
              "%s: too many output tiles", what);
  const unsigned blocks = static_cast<unsigned>(grid < most ? grid : most);
  lin_tile_kernel<OP, KIND, FQ, FP, STAGED><<<blocks, 512, 0, s>>>(a, pl);
  return check_launch(what);
}

template <int OP, int KIND, int FQ, int FP, bool STAGED>
int launch_rows(const LinArgs& a, hipStream_t s, const char* what) {
  const int64_t grid = lin_tile_grid(a, 64 * FQ, 128 * FP);
  return launch<OP, KIND, FQ, FP, STAGED>(a, LinPlanArgs{}, grid, s, what);
}

template <int OP, int KIND>
int pick_rows(const LinArgs& a, LinTileShape t, hipStream_t s, const char* what) {
  if (t.staged) {
    if (t.rows >= 128) return launch_rows<OP, KIND, 2, 2, true>(a, s, what);
    return t.cols == 256 ? launch_rows<OP, KIND, 1, 2, true>(a, s, what)
                         : launch_rows<OP, KIND, 1, 1, true>(a, s, what);
  }
  if (t.rows == 256) return launch_rows<OP, KIND, 4, 2, false>(a, s, what);
  if (t.rows == 128) return launch_rows<OP, KIND, 2, 2, false>(a, s, what);
  return t.cols == 256 ? launch_rows<OP, KIND, 1, 2, false>(a, s, what)
                       : launch_rows<OP, KIND, 1, 1, false>(a, s, what);
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
    default: return pick_rows<kOpMx8, kLinForward>(a, t, s, what);
  }
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
