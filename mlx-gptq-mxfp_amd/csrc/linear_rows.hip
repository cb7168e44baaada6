// Row operators beside the matrix products: quantizing rows to 8-bit integers,
// and the sum of list entries per row that ends a gathered product's gradient.
#include "linear_common.h"

namespace mgq {
namespace {

// ---------------------------------------------------------------------------
// q = round-half-even(x / s), s = max|x| / 127, both IEEE fp32 quotients, |q| <=
// 127. A zero row has s = 0 and q = 0; a row that holds a NaN or an infinity has
// s = NaN and q = 0, so that every product with it is NaN.
//
// Bound by memory (65537 x 5120 bf16 in 0.17 ms, 5.8 TB/s read and written): a row
// is read once and stays in registers, PIECES of 16 bytes a lane, between its
// maximum and its codes; WAVES waves share it. Longer rows (PIECES = 0) are read
// twice. Rows have any pitch and alignment: a 16-byte load takes any address, and
// the piece a row ends in is read element by element.
//
// Codes: with y = RN(1 / s), q = fma(fma(-x y, s, x), y, x y) is the IEEE quotient
// x / s wherever s is in [2^-24, 2^24] and the quotient is not tiny (where it
// rounds to 0 all the same); adding 1.5 2^23 rounds it half-even to an integer
// whose low byte is the code. Rows with other scales divide.
// ---------------------------------------------------------------------------
struct __attribute__((packed, aligned(1))) u64_u_t {
  uint32_t v[2];
};

template <int DT>
struct RowPiece {
  static constexpr int N = DT == kF32 ? 4 : 8;  // elements
  lin_u32x4_t v;

  __device__ __forceinline__ void load(const char* row, int64_t c, int64_t cols) {
    constexpr int ES = 16 / N;
    v = lin_u32x4_t{0, 0, 0, 0};
    if (c + N <= cols) {
      const lin_u128_u_t u = *reinterpret_cast<const lin_u128_u_t*>(row + c * ES);
      v = lin_u32x4_t{u.v[0], u.v[1], u.v[2], u.v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < cols) {
          if constexpr (DT == kF32)
            v[i] = *reinterpret_cast<const uint32_t*>(row + (c + i) * 4);
          else
            v[i >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row + (c + i) * 2))
                         << (16 * (i & 1));
        }
    }
  }
  // |x| as bits, which order like the values (NaN and infinity above all): fp32 in
  // one maximum, 16-bit types in two 16-bit ones
  __device__ __forceinline__ void bits_max(uint32_t& m) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kF32) {
        const uint32_t u = v[i] & 0x7fffffffu;
        m = m > u ? m : u;
      } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        const u16x2 x = __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu);
        const u16x2 o = __builtin_bit_cast(u16x2, m);
        m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, o));
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (DT == kF32) return u2f(v[i]);
    const uint32_t w = v[i >> 1];
    if constexpr (DT == kBF16) return u2f(i & 1 ? w & 0xffff0000u : w << 16);
    return f16_to_f32(static_cast<uint16_t>(i & 1 ? w >> 16 : w));
  }
};

template <int DT, int WAVES, int PIECES>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const char* __restrict__ X, int64_t n_rows, int64_t cols, int64_t ldx,
                         int8_t* __restrict__ q, float* __restrict__ scales) {
  typedef RowPiece<DT> piece_t;
  constexpr int N = piece_t::N, T = 64 * WAVES, ROWS = 4 / WAVES;
  __shared__ uint32_t part[4];
  const int t = threadIdx.x % T;
  const int64_t row = blockIdx.x * static_cast<int64_t>(ROWS) + threadIdx.x / T;
  if (WAVES == 1 && row >= n_rows) return;
  const char* x = X + row * ldx * (16 / N);
  piece_t keep[PIECES > 0 ? PIECES : 1];
  uint32_t m = 0;
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) keep[i].load(x, (static_cast<int64_t>(i) * T + t) * N, cols);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) keep[i].bits_max(m);
  } else {
    for (int64_t c = static_cast<int64_t>(t) * N; c < cols; c += T * N) {
      keep[0].load(x, c, cols);
      keep[0].bits_max(m);
    }
  }
  if constexpr (DT != kF32) m = m >> 16 > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = __shfl_xor(m, d);
    m = m > o ? m : o;
  }
  if constexpr (WAVES == 4) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) m = m > part[i] ? m : part[i];
  }
  const float amax = DT == kF32 ? u2f(m) : DT == kBF16 ? u2f(m << 16) : f16_to_f32(m);
  const bool bad = !(amax <= 3.40282347e38f);
  const float s = bad ? u2f(0x7fc00000u) : amax / 127.0f;
  if (t == 0) scales[row] = s;
  const bool plain = s >= 5.96046448e-8f && s <= 16777216.0f;
  const float y = plain ? 1.0f / s : 0.0f;
  auto store = [&](const piece_t& p, int64_t c) {
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = p.get(i);
      float r;
      if (plain) {
        const float g = v * y;
        r = fmaf(fmaf(-g, s, v), y, g);
      } else {
        r = !bad && s > 0.0f ? fminf(fmaxf(v / s, -127.0f), 127.0f) : 0.0f;
      }
      b[i] = f2u(r + 12582912.0f);
    }
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000c0cu);
      w[i] = lo | hi;
    }
    int8_t* o = q + row * cols + c;
    if (c + N <= cols) {
      if constexpr (N == 8) {
        u64_u_t u;
        u.v[0] = w[0];
        u.v[1] = w[1];
        *reinterpret_cast<u64_u_t*>(o) = u;
      } else {
        struct __attribute__((packed, aligned(1))) u32_u_t { uint32_t v; } u = {w[0]};
        *reinterpret_cast<u32_u_t*>(o) = u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c + i < cols) o[i] = static_cast<int8_t>(b[i]);
    }
  };
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) store(keep[i], (static_cast<int64_t>(i) * T + t) * N);
  } else {
    for (int64_t c = static_cast<int64_t>(t) * N; c < cols; c += T * N) {
      keep[0].load(x, c, cols);
      store(keep[0], c);
    }
  }
}

// Rows of one launch: a workgroup a row has 256 threads, a launch less than 2^32.
constexpr int64_t kLaunchRows = int64_t(1) << 23;

// A wave per row while four pieces a lane hold it, then a workgroup.
template <int DT>
void quantize_rows(const char* X, int64_t n_rows, int64_t cols, int64_t ldx, int8_t* q,
                   float* scales, hipStream_t s) {
  const int64_t pieces = ceil_div(cols, RowPiece<DT>::N);
  for (int64_t r0 = 0; r0 < n_rows; r0 += kLaunchRows) {
    const int64_t rows = n_rows - r0 < kLaunchRows ? n_rows - r0 : kLaunchRows;
    const unsigned quads = static_cast<unsigned>(ceil_div(rows, 4)), wg = static_cast<unsigned>(rows);
    const char* x = X + r0 * ldx * (16 / RowPiece<DT>::N);
    int8_t* qr = q + r0 * cols;
    float* sr = scales + r0;
    if (pieces <= 64)
      quantize_rows_kernel<DT, 1, 1><<<quads, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else if (pieces <= 128)
      quantize_rows_kernel<DT, 1, 2><<<quads, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else if (pieces <= 256)
      quantize_rows_kernel<DT, 1, 4><<<quads, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else if (pieces <= 512)
      quantize_rows_kernel<DT, 4, 2><<<wg, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else if (pieces <= 768)
      quantize_rows_kernel<DT, 4, 3><<<wg, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else if (pieces <= 1024)
      quantize_rows_kernel<DT, 4, 4><<<wg, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else if (pieces <= 2048)
      quantize_rows_kernel<DT, 4, 8><<<wg, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
    else
      quantize_rows_kernel<DT, 4, 0><<<wg, 256, 0, s>>>(x, rows, cols, ldx, qr, sr);
  }
}

// ---------------------------------------------------------------------------
// out[r] = sum of src[t] over the list entries t with row_index[t] = r, in the
// order of t, in fp32. The entries of a row arrive in any order: the first kSlots
// take its slots, the others chain up behind its head, and the sum sorts them, so
// that it does not depend on the atomics' order. A row of n entries past its slots
// walks its chain once for every 64 of them, keeping the next 64 in order over the
// lanes, or reads the whole list, 64 indexes at a time, where that is less: the
// loads that wait for each other are at most n^2 / 64 and M / 64, together M^1.5 / 64
// for any list. Bound by memory: 8198 entries into 4099 rows of 1024 take 8.2 us (50 MB,
// mostly from the caches), and clearing and filling the slots 3 us each; both in one
// workgroup took 16. 16384 rows of 64 read 24 times each take 0.18 ms with the product
// in front, read 16 times each 0.12.
// ---------------------------------------------------------------------------
constexpr int kSlots = 16;
constexpr int kSumCols = 1024;  // columns a wave sums at once

struct RowState {
  int32_t count;  // entries
  int32_t head;   // the last one that found no slot, -1 if all did
};

__global__ void __launch_bounds__(256) rows_clear_kernel(RowState* __restrict__ state, int64_t n) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
    state[i] = RowState{0, -1};
}

__device__ inline int64_t clamp_row(int64_t r, int64_t n_rows) {
  r = r < 0 ? 0 : r;
  return r < n_rows ? r : n_rows - 1;
}

__global__ void __launch_bounds__(256)
    rows_fill_kernel(const int32_t* __restrict__ row_index, int64_t M, int64_t n_rows,
                     RowState* __restrict__ state, int32_t* __restrict__ slots,
                     int32_t* __restrict__ next) {
  for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < M; t += gridDim.x * 256ll) {
    const int64_t r = clamp_row(row_index[t], n_rows);
    const int32_t i = atomicAdd(&state[r].count, 1);
    if (i < kSlots)
      slots[r * kSlots + i] = static_cast<int32_t>(t);
    else
      next[t] = atomicExch(&state[r].head, static_cast<int32_t>(t));
  }
}

__global__ void __launch_bounds__(256)
    rows_sum_kernel(const float* __restrict__ src, const int32_t* __restrict__ row_index, int64_t M,
                    int64_t first, int64_t n_rows, int64_t cols,
                    const RowState* __restrict__ state, const int32_t* __restrict__ slots,
                    const int32_t* __restrict__ next, void* __restrict__ out, int out_type) {
  const int lane = threadIdx.x & 63;
  const int64_t r = first + blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (r >= n_rows) return;
  const int n = __builtin_amdgcn_readfirstlane(state[r].count);
  const int head = __builtin_amdgcn_readfirstlane(state[r].head);
  const bool chained = n > kSlots && (n + 63ll) / 64 * n <= M / 64;
  // lane k: entry k in the list's order (up to kSlots), or slot k
  const int32_t slot = lane < (n < kSlots ? n : kSlots) ? slots[r * kSlots + lane] : 0;
  int32_t mine = 0;
  if (n <= kSlots) {
    int rank = lane < n ? 0 : lane;
    for (int j = 0; j < n; ++j) rank += (lane < n && __builtin_amdgcn_readlane(slot, j) < slot) ? 1 : 0;
    mine = __builtin_amdgcn_ds_permute(4 * rank, slot);
  }
  // the 64 smallest entries above `last` (a chain has n - kSlots entries)
  auto next_batch = [&](int32_t last) {
    int32_t best = 0x7fffffff;
    auto insert = [&](int32_t t) {
      if (t <= last) return;
      const int at = static_cast<int>(__popcll(__ballot(best < t)));
      const int32_t below = __shfl_up(best, 1);
      best = lane > at ? below : lane == at ? t : best;
    };
    for (int j = 0; j < kSlots; ++j) insert(__builtin_amdgcn_readlane(slot, j));
    int32_t t = head;
    for (int k = kSlots; k < n && t >= 0; ++k) {
      const int32_t after = __builtin_amdgcn_readfirstlane(next[t]);
      insert(t);
      t = after;
    }
    return best;
  };
  for (int64_t c0 = 0; c0 < cols; c0 += kSumCols) {
    // four consecutive columns a lane and piece
    constexpr int kPieces = kSumCols / 256;
    f32x4_u_t acc[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) acc[i] = f32x4_u_t{0, 0, 0, 0};
    auto add = [&](int64_t t) {
      const float* p = src + t * cols + c0 + 4 * lane;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int64_t c = c0 + 256 * i + 4 * lane;
        if (c + 4 <= cols) {
          acc[i] += load_f32x4(p + 256 * i);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < cols) acc[i][e] += p[256 * i + e];
        }
      }
    };
    if (n <= kSlots) {
      for (int j = 0; j < n; ++j) add(__builtin_amdgcn_readlane(mine, j));
    } else if (chained) {
      int32_t last = -1;
      for (int done = 0; done < n; done += 64) {
        const int32_t batch = next_batch(last);
        const int m = n - done < 64 ? n - done : 64;
        for (int j = 0; j < m; ++j) add(__builtin_amdgcn_readlane(batch, j));
        last = __builtin_amdgcn_readlane(batch, m - 1);
      }
    } else {
      for (int64_t t0 = 0; t0 < M; t0 += 64) {
        const bool hit = t0 + lane < M && clamp_row(row_index[t0 + lane], n_rows) == r;
        for (uint64_t b = __ballot(hit); b; b &= b - 1) add(t0 + __builtin_ctzll(b));
      }
    }
    LinArgs a = {};  // lin_store4's row length and type
    a.np = static_cast<int>(cols);
    a.out_type = out_type;
    char* row = static_cast<char*>(out) + r * cols * (out_type == kF32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int64_t c = c0 + 256 * i + 4 * lane;
      const float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
      if (c < cols) lin_store4(a, row, static_cast<int>(c), v);
    }
  }
}

int64_t pad256(int64_t n) { return ceil_div(n, 256) * 256; }
// workspace: the rows' states, their slots, the entries' chain
int64_t slots_off(int64_t n_rows) { return pad256(n_rows * static_cast<int64_t>(sizeof(RowState))); }
int64_t next_off(int64_t n_rows) { return slots_off(n_rows) + pad256(4 * kSlots * n_rows); }

}  // namespace
}  // namespace mgq

using namespace mgq;

extern "C" int mgq_quantize_rows_int8(const void* X, int dtype, int64_t rows, int64_t cols,
                                      int64_t ldx, int8_t* q, float* scales, void* stream) {
  clear_error();
  MGQ_REQUIRE(dtype == kF32 || dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE,
              "quantize_rows_int8: float32, bfloat16 or float16 only");
  MGQ_REQUIRE(rows >= 0 && cols >= 1 && ldx >= cols && rows < (int64_t(1) << 31), MGQ_ERR_SHAPE,
              "quantize_rows_int8: bad shape [%lld, %lld]", (long long)rows, (long long)cols);
  if (rows == 0) return MGQ_OK;
  const char* x = static_cast<const char*>(X);
  hipStream_t st = as_stream(stream);
  if (dtype == kF32)
    quantize_rows<kF32>(x, rows, cols, ldx, q, scales, st);
  else if (dtype == kBF16)
    quantize_rows<kBF16>(x, rows, cols, ldx, q, scales, st);
  else
    quantize_rows<kF16>(x, rows, cols, ldx, q, scales, st);
  return check_launch("quantize_rows_int8");
}

extern "C" int64_t mgq_rows_sum_workspace_size(int64_t n_entries, int64_t n_rows) {
  return n_entries < 0 || n_rows < 0 ? 0 : next_off(n_rows) + 4 * n_entries;
}

extern "C" int mgq_rows_sum(const float* src, const int32_t* row_index, int64_t n_entries,
                            int64_t n_rows, int64_t cols, void* out, int out_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  clear_error();
  MGQ_REQUIRE(out_dtype == kF32 || out_dtype == kBF16 || out_dtype == kF16, MGQ_ERR_VALUE,
              "rows_sum: the result is float32, bfloat16 or float16");
  MGQ_REQUIRE(n_entries >= 0 && n_entries < (int64_t(1) << 31) && n_rows >= 0 &&
                  n_rows < (int64_t(1) << 31) && cols >= 0 && cols < (int64_t(1) << 30),
              MGQ_ERR_SHAPE, "rows_sum: bad shape");
  const int64_t need = mgq_rows_sum_workspace_size(n_entries, n_rows);
  MGQ_REQUIRE(workspace != nullptr && workspace_bytes >= need, MGQ_ERR_WORKSPACE,
              "rows_sum workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  if (n_rows == 0 || cols == 0) return MGQ_OK;
  hipStream_t s = as_stream(stream);
  char* ws = static_cast<char*>(workspace);
  RowState* state = reinterpret_cast<RowState*>(ws);
  int32_t* slots = reinterpret_cast<int32_t*>(ws + slots_off(n_rows));
  int32_t* next = reinterpret_cast<int32_t*>(ws + next_off(n_rows));
  rows_clear_kernel<<<elementwise_blocks(n_rows, 256), 256, 0, s>>>(state, n_rows);
  if (n_entries > 0)
    rows_fill_kernel<<<elementwise_blocks(n_entries, 256), 256, 0, s>>>(row_index, n_entries, n_rows,
                                                                        state, slots, next);
  for (int64_t r0 = 0; r0 < n_rows; r0 += kLaunchRows) {
    const int64_t rows = n_rows - r0 < kLaunchRows ? n_rows - r0 : kLaunchRows;
    rows_sum_kernel<<<static_cast<unsigned>(ceil_div(rows, 4)), 256, 0, s>>>(
        src, row_index, n_entries, r0, n_rows, cols, state, slots, next, out, out_dtype);
  }
  return check_launch("rows_sum");
}
