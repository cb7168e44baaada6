// Matrix products grouped by expert: dense (bf16, f16), MXFP4 / MXFP8 and int8
// weights; both gradients of the dense form. Group g owns the list entries
// [offsets[g], offsets[g + 1]); entry t reads row row_index[t] of X (or row t).
//
// linear_any_kernel takes every size, pitch and alignment: operands go
// through registers into LDS, piecewise where a row ends inside a 16-byte
// piece.
#include "linear_tile.h"

namespace mgq {
namespace {

constexpr int kAnyT = 128;     // output tile 128 x 128
constexpr int kAnyB = 64;      // bytes of a row per stage: 32 16-bit or 64 int8 elements
constexpr int kAnyPitch = 80;  // LDS row pitch, 16-byte aligned

// 16 bytes of a row: `n` of its elements exist, the rest are zeros.
template <int ES>
__device__ __forceinline__ lin_u32x4_t load_piece(const char* p, int n) {
  lin_u32x4_t r = {0, 0, 0, 0};
  if (n >= 16 / ES) {
    const lin_u128_u_t u = *reinterpret_cast<const lin_u128_u_t*>(p);
    r = lin_u32x4_t{u.v[0], u.v[1], u.v[2], u.v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 16 / ES; ++i) {
      if (i < n) {
        const uint32_t v = ES == 2 ? *reinterpret_cast<const uint16_t*>(p + 2 * i)
                                   : *reinterpret_cast<const uint8_t*>(p + i);
        r[i * ES / 4] |= v << (8 * ((i * ES) & 3));
      }
    }
  }
  return r;
}

// Piece c (16 bytes of bf16, i.e. 8 elements) of an MX weight row.
template <int OP>
__device__ __forceinline__ lin_u32x4_t load_mx_piece(const char* row, const uint8_t* srow, int c0,
                                                     int nc) {
  lin_u32x4_t r = {0, 0, 0, 0};
  if (c0 < nc) {  // nc is a multiple of 32
    const uint32_t s = srow[c0 >> 5];
    if constexpr (OP == kOpMx4) {
      r = lin_decode_mx4(*reinterpret_cast<const uint32_t*>(row + (c0 >> 1)), s);
    } else {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(row + c0);
      r = lin_decode_mx8(q[0], q[1], s);
    }
  }
  return r;
}

// PT / QT: the operand's contraction dimension is its row dimension
// (transposed reads, 16-bit types only). RAGGED_C: wgrad, whose contraction
// runs over a group's entries.
template <int OP, bool PT, bool QT, bool RAGGED_C>
__global__ void __launch_bounds__(256) linear_any_kernel(const LinArgs a) {
  constexpr int ES = lin_esize<OP>();
  constexpr int EP = 16 / ES;         // elements per piece
  constexpr int EK = kAnyB / ES;      // contraction elements per stage
  typedef typename LinAcc<OP>::t32 acc_t;
  __shared__ __attribute__((aligned(16))) char lds[2 * kAnyT * kAnyPitch];
  char* lq = lds;
  char* lp = lds + kAnyT * kAnyPitch;

  int g, p0, q0, nq;
  int64_t c_begin = 0, c_end = a.nc;  // contraction range
  int64_t e0 = 0;                     // forward, dgrad: list entry of q = 0
  if constexpr (RAGGED_C) {
    const int npt = (a.np + kAnyT - 1) / kAnyT, nqt = (a.nq + kAnyT - 1) / kAnyT;
    const uint32_t per = static_cast<uint32_t>(npt) * nqt;
    g = blockIdx.x / per;
    const uint32_t in = blockIdx.x % per;
    p0 = (in % npt) * kAnyT;
    q0 = (in / npt) * kAnyT;
    nq = a.nq;
    c_end = a.M;
    if (a.offsets) lin_segment(a, g, &c_begin, &c_end);
    if (c_end < c_begin) c_end = c_begin;
  } else {
    LinTile t;
    if (!lin_find_tile<kAnyT>(a, (a.np + kAnyT - 1) / kAnyT, &t)) return;
    g = t.g;
    p0 = t.pt * kAnyT;
    q0 = 0;
    e0 = t.q0;
    nq = static_cast<int>(t.q_end - t.q0 < kAnyT ? t.q_end - t.q0 : kAnyT);
    if (g >= a.G) c_end = 0;  // entries of no group: zeros
  }

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wq = (wave >> 1) * 64, wp = (wave & 1) * 64;
  const int gw = RAGGED_C || g >= a.G ? 0 : g;
  const char* Pg = a.P + gw * a.p_group;
  const uint8_t* Psg =
      lin_is_mx<OP>() ? a.Ps + static_cast<int64_t>(gw) * a.np * (a.nc / 32) : nullptr;

  lin_u32x4_t rq[2], rp[2];
  // thread's pieces: plain operands by (row, piece of 4), transposed ones by
  // (contraction row of 32, 8 columns of 128)
  auto fetch = [&](int64_t c0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int id = tid + 256 * j;
      rq[j] = lin_u32x4_t{0, 0, 0, 0};
      rp[j] = lin_u32x4_t{0, 0, 0, 0};
      if constexpr (QT) {
        const int64_t c = c0 + (id >> 4);
        const int col = q0 + 8 * (id & 15);
        if (c < c_end && col < a.nq) rq[j] = load_piece<ES>(a.Q + c * a.ldq + 2 * col, a.nq - col);
      } else {
        const int r = id >> 2;
        const int64_t c = c0 + (id & 3) * EP;
        if (r < nq && c < c_end) {
          const int64_t row = PT ? e0 + r : lin_row(a, e0 + r);
          rq[j] = load_piece<ES>(a.Q + row * a.ldq + c * ES,
                                 static_cast<int>(c_end - c < EP ? c_end - c : EP));
        }
      }
      if constexpr (PT) {
        const int64_t c = c0 + (id >> 4);
        const int col = p0 + 8 * (id & 15);
        if (c < c_end && col < a.np) {
          const int64_t row = RAGGED_C ? lin_row(a, c) : c;
          rp[j] = load_piece<ES>(Pg + row * a.ldp + 2 * col, a.np - col);
        }
      } else {
        const int p = p0 + (id >> 2);
        const int64_t c = c0 + (id & 3) * EP;
        if (p < a.np && c < c_end) {
          if constexpr (lin_is_mx<OP>())
            rp[j] = load_mx_piece<OP>(Pg + p * a.ldp, Psg + static_cast<int64_t>(p) * (a.nc / 32),
                                      static_cast<int>(c), a.nc);
          else
            rp[j] = load_piece<ES>(Pg + p * a.ldp + c * ES,
                                   static_cast<int>(c_end - c < EP ? c_end - c : EP));
        }
      }
    }
  };
  auto put = [&](char* l, bool transposed, lin_u32x4_t v, int id) {
    if (transposed) {
      const int c = id >> 4, r = 8 * (id & 15);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint16_t*>(l + (r + i) * kAnyPitch + 2 * c) =
            static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
    } else {
      *reinterpret_cast<lin_u32x4_t*>(l + (id >> 2) * kAnyPitch + 16 * (id & 3)) = v;
    }
  };

  acc_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

  if (c_begin < c_end) fetch(c_begin);
  for (int64_t c = c_begin; c < c_end; c += EK) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      put(lq, QT, rq[j], tid + 256 * j);
      put(lp, PT, rp[j], tid + 256 * j);
    }
    __syncthreads();
    if (c + EK < c_end) fetch(c + EK);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int off = (2 * ks + (lane >> 5)) * 16;
      lin_u32x4_t fp[2], fq[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fp[i] = *reinterpret_cast<const lin_u32x4_t*>(
            lp + (wp + 32 * i + (lane & 31)) * kAnyPitch + off);
        fq[i] = *reinterpret_cast<const lin_u32x4_t*>(
            lq + (wq + 32 * i + (lane & 31)) * kAnyPitch + off);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = lin_mfma32<OP>(fp[i], fq[j], acc[i][j]);
    }
  }

  const int osize = a.out_type == kF32 ? 4 : 2;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int q = q0 + wq + 32 * j + (lane & 31);
    if (q >= nq) continue;
    const int64_t orow = RAGGED_C ? q : e0 + q;
    char* row = a.out + (orow * a.ldo + (RAGGED_C ? g * a.o_group : 0)) * osize;
    float sx = 0.0f;
    if constexpr (OP == kOpI8) sx = g < a.G ? a.sx[lin_row(a, e0 + q)] : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = p0 + wp + 32 * i + 8 * r + 4 * (lane >> 5);
        if (p >= a.np) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(acc[i][j][4 * r + e]);
        if (g < a.G) lin_scale4<OP>(a, g, p, sx, v);
        lin_store4(a, row, p, v);
      }
  }
}

template <int OP, bool PT, bool QT, bool RC>
int launch_any(const LinArgs& a, int64_t grid, hipStream_t s, const char* what) {
  MGQ_REQUIRE(grid < (int64_t(1) << 31), MGQ_ERR_SHAPE, "%s: too many output tiles", what);
  linear_any_kernel<OP, PT, QT, RC><<<static_cast<unsigned>(grid), 256, 0, s>>>(a);
  return check_launch(what);
}

// Forward and dgrad. The large tiles take operands of whole 16-byte pieces; how
// many rows a tile has goes by the average group's.
template <int OP, int KIND>
int run_rows(const LinArgs& a, hipStream_t s, const char* what) {
  if (lin_tile_takes(a, OP, KIND)) {
    const int64_t avg = a.M / a.G;
    return lin_tile_rows(a, OP, KIND, avg > 192 ? 4 : avg > 64 ? 2 : 1, s, what);
  }
  const int64_t grid = lin_row_tiles(a, kAnyT) * ceil_div(a.np, kAnyT);
  return launch_any<OP, KIND == kLinDgrad, false, false>(a, grid, s, what);
}

int check_list(const char* what, const int32_t* offsets, const int32_t* row_index,
               int64_t n_groups, int64_t n_entries, int64_t n_rows) {
  MGQ_REQUIRE(n_groups >= 1 && n_groups <= (int64_t(1) << 20), MGQ_ERR_SHAPE,
              "%s: %lld groups (1 .. 2^20)", what, (long long)n_groups);
  MGQ_REQUIRE(offsets != nullptr || n_groups == 1, MGQ_ERR_VALUE,
              "%s: offsets required for %lld groups", what, (long long)n_groups);
  MGQ_REQUIRE(n_entries >= 0 && n_entries < (int64_t(1) << 31) - 4096, MGQ_ERR_SHAPE,
              "%s: %lld list entries", what, (long long)n_entries);
  MGQ_REQUIRE(n_rows >= 1 || n_entries == 0, MGQ_ERR_SHAPE, "%s: X has no rows", what);
  MGQ_REQUIRE(row_index != nullptr || n_entries <= n_rows, MGQ_ERR_SHAPE,
              "%s: %lld list entries but X has %lld rows", what, (long long)n_entries,
              (long long)n_rows);
  return MGQ_OK;
}

int check_dims(const char* what, int64_t N, int64_t K) {
  MGQ_REQUIRE(N >= 1 && K >= 0 && N < (int64_t(1) << 30) && K < (int64_t(1) << 30), MGQ_ERR_SHAPE,
              "%s: bad weight shape [%lld, %lld]", what, (long long)N, (long long)K);
  return MGQ_OK;
}

// 2: 16-byte stores, 1: four results at once, 0: one by one.
int vec_ok(const void* out, int64_t ldo, int out_type) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(out);
  if (ldo % 8 == 0 && (at & 15) == 0) return 2;
  return ldo % 4 == 0 && (at & (out_type == kF32 ? 15 : 7)) == 0;
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
  if (int rc = check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = check_dims(what, N, K)) return rc;
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
  a.vec_out = vec_ok(Y, N, dtype);
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
  if (int rc = check_list(what, offsets, nullptr, n_groups, n_entries, n_entries)) return rc;
  if (int rc = check_dims(what, N, K)) return rc;
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
  a.vec_out = vec_ok(dX, K, out_dtype);
  hipStream_t s = as_stream(stream);
  return dtype == kF16 ? run_rows<kOpF16, kLinDgrad>(a, s, what)
                       : run_rows<kOpBF16, kLinDgrad>(a, s, what);
}

extern "C" int64_t mgq_grouped_wgrad_workspace_size(int64_t n_entries, int64_t n_groups, int64_t N,
                                                    int64_t K) {
  if (n_entries < 0 || n_groups < 1 || n_groups > kLinPlanGroups || N < 1 || K < 1) return 0;
  return lin_plan_sizes(n_entries, n_groups, N, K).bytes;
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
  if (int rc = check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = check_dims(what, N, K)) return rc;
  MGQ_REQUIRE(lddy >= N && ldx >= K, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
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
  a.vec_out = vec_ok(dW, K, out_dtype);
  hipStream_t s = as_stream(stream);
  if (lin_tile_takes(a, dtype == kF16 ? kOpF16 : kOpBF16, kLinWgrad))
    return lin_tile_wgrad(a, dtype == kF16 ? kOpF16 : kOpBF16, workspace, s, what);
  const int64_t grid = n_groups * ceil_div(N, kAnyT) * ceil_div(K, kAnyT);
  return dtype == kF16 ? launch_any<kOpF16, true, true, true>(a, grid, s, what)
                       : launch_any<kOpBF16, true, true, true>(a, grid, s, what);
}

extern "C" int mgq_mxfp_linear(const void* X, int64_t n_rows, int64_t ldx, const int32_t* row_index,
                               int64_t n_entries, const uint32_t* words, const uint8_t* scales,
                               int mode, int64_t n_groups, int64_t N, int64_t K,
                               const int32_t* offsets, void* Y, void* stream) {
  clear_error();
  const char* what = "mxfp_linear";
  MGQ_REQUIRE(mode == kMxfp4 || mode == kMxfp8, MGQ_ERR_VALUE, "%s: mode must be mxfp4 or mxfp8",
              what);
  if (int rc = check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = check_dims(what, N, K)) return rc;
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
  a.vec_out = vec_ok(Y, N, kBF16);
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
  if (int rc = check_list(what, offsets, row_index, n_groups, n_entries, n_rows)) return rc;
  if (int rc = check_dims(what, N, K)) return rc;
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
  a.vec_out = vec_ok(Y, N, out_dtype);
  a.sx = x_scale;
  a.sw = w_scale;
  a.bias = bias;
  return run_rows<kOpI8, kLinForward>(a, as_stream(stream), what);
}
