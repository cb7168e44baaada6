// Row operators beside the matrix products: quantizing rows to 8-bit integers,
// and the sum of list entries per row that ends a gathered product's gradient.
#include "linear_common.h"

namespace mgq {
namespace {

// ---------------------------------------------------------------------------
// q = round-half-even(x / s), s = max|x| / 127, both IEEE fp32 quotients. A
// zero row has s = 0 and q = 0; a row that holds a NaN or an infinity has
// s = NaN and q = 0, so that every product with it is NaN.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const char* __restrict__ X, int dtype, int64_t cols, int64_t ldx,
                         int8_t* __restrict__ q, float* __restrict__ scales) {
  __shared__ uint32_t part[4];
  const int64_t row = blockIdx.x;
  const char* x = X + row * ldx * (dtype == kF32 ? 4 : 2);
  uint32_t m = 0;  // |x| as bits: NaN and infinity order above every finite value
  for (int64_t c = threadIdx.x; c < cols; c += 256) {
    const uint32_t u = f2u(load_storage(x, c, dtype)) & 0x7fffffffu;
    m = m > u ? m : u;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = __shfl_xor(m, d);
    m = m > o ? m : o;
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m = m > part[i] ? m : part[i];
  const bool bad = m >= 0x7f800000u;
  const float s = bad ? u2f(0x7fc00000u) : u2f(m) / 127.0f;
  if (threadIdx.x == 0) scales[row] = s;
  for (int64_t c = threadIdx.x; c < cols; c += 256) {
    float v = 0.0f;
    if (!bad && s > 0.0f) v = fminf(fmaxf(rintf(load_storage(x, c, dtype) / s), -127.0f), 127.0f);
    q[row * cols + c] = static_cast<int8_t>(v);
  }
}

// ---------------------------------------------------------------------------
// out[r] = sum of src[t] over the list entries t with row_index[t] = r, in the
// order of t, in fp32. Each row has kSlots slots that the entries fill in any
// order; the sum sorts them, so it does not depend on the atomics' order. A row
// with more entries than slots finds them by scanning the list.
// ---------------------------------------------------------------------------
constexpr int kSlots = 16;
constexpr int kSumCols = 1024;  // columns a wave sums at once

__global__ void __launch_bounds__(256) rows_clear_kernel(int32_t* __restrict__ count, int64_t n) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) count[i] = 0;
}

__device__ inline int64_t clamp_row(int64_t r, int64_t n_rows) {
  r = r < 0 ? 0 : r;
  return r < n_rows ? r : n_rows - 1;
}

__global__ void __launch_bounds__(256)
    rows_fill_kernel(const int32_t* __restrict__ row_index, int64_t M, int64_t n_rows,
                     int32_t* __restrict__ count, int32_t* __restrict__ slots) {
  for (int64_t t = blockIdx.x * 256ll + threadIdx.x; t < M; t += gridDim.x * 256ll) {
    const int64_t r = clamp_row(row_index[t], n_rows);
    const int32_t i = atomicAdd(&count[r], 1);
    if (i < kSlots) slots[r * kSlots + i] = static_cast<int32_t>(t);
  }
}

__global__ void __launch_bounds__(256)
    rows_sum_kernel(const float* __restrict__ src, const int32_t* __restrict__ row_index, int64_t M,
                    int64_t n_rows, int64_t cols, const int32_t* __restrict__ count,
                    const int32_t* __restrict__ slots, void* __restrict__ out, int out_type) {
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (r >= n_rows) return;
  const int n = __builtin_amdgcn_readfirstlane(count[r]);
  int32_t mine = 0;
  if (n <= kSlots) {
    const int32_t v = lane < n ? slots[r * kSlots + lane] : 0;
    int rank = lane < n ? 0 : lane;
    for (int j = 0; j < n; ++j) rank += (lane < n && __builtin_amdgcn_readlane(v, j) < v) ? 1 : 0;
    mine = __builtin_amdgcn_ds_permute(4 * rank, v);
  }
  for (int64_t c0 = 0; c0 < cols; c0 += kSumCols) {
    float acc[kSumCols / 64];
#pragma unroll
    for (int i = 0; i < kSumCols / 64; ++i) acc[i] = 0.0f;
    auto add = [&](int64_t t) {
      const float* p = src + t * cols + c0;
#pragma unroll
      for (int i = 0; i < kSumCols / 64; ++i)
        if (c0 + 64 * i + lane < cols) acc[i] += p[64 * i + lane];
    };
    if (n <= kSlots) {
      for (int j = 0; j < n; ++j) add(__builtin_amdgcn_readlane(mine, j));
    } else {
      for (int64_t t0 = 0; t0 < M; t0 += 64) {
        const bool hit = t0 + lane < M && clamp_row(row_index[t0 + lane], n_rows) == r;
        for (uint64_t b = __ballot(hit); b; b &= b - 1) add(t0 + __builtin_ctzll(b));
      }
    }
#pragma unroll
    for (int i = 0; i < kSumCols / 64; ++i)
      if (c0 + 64 * i + lane < cols) store_storage(out, r * cols + c0 + 64 * i + lane, acc[i], out_type);
  }
}

int64_t slots_off(int64_t n_rows) { return ceil_div(4 * n_rows, 256) * 256; }

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
  quantize_rows_kernel<<<static_cast<unsigned>(rows), 256, 0, as_stream(stream)>>>(
      static_cast<const char*>(X), dtype, cols, ldx, q, scales);
  return check_launch("quantize_rows_int8");
}

extern "C" int64_t mgq_rows_sum_workspace_size(int64_t n_rows) {
  return slots_off(n_rows) + 4 * kSlots * n_rows;
}

extern "C" int mgq_rows_sum(const float* src, const int32_t* row_index, int64_t n_entries,
                            int64_t n_rows, int64_t cols, void* out, int out_dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  clear_error();
  MGQ_REQUIRE(out_dtype == kF32 || out_dtype == kBF16 || out_dtype == kF16, MGQ_ERR_VALUE,
              "rows_sum: the result is float32, bfloat16 or float16");
  MGQ_REQUIRE(n_entries >= 0 && n_entries < (int64_t(1) << 31) && n_rows >= 0 &&
                  n_rows < (int64_t(1) << 31) && cols >= 0,
              MGQ_ERR_SHAPE, "rows_sum: bad shape");
  const int64_t need = mgq_rows_sum_workspace_size(n_rows);
  MGQ_REQUIRE(workspace != nullptr && workspace_bytes >= need, MGQ_ERR_WORKSPACE,
              "rows_sum workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  if (n_rows == 0 || cols == 0) return MGQ_OK;
  hipStream_t s = as_stream(stream);
  int32_t* count = static_cast<int32_t*>(workspace);
  int32_t* slots = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + slots_off(n_rows));
  rows_clear_kernel<<<elementwise_blocks(n_rows, 256), 256, 0, s>>>(count, n_rows);
  if (n_entries > 0)
    rows_fill_kernel<<<elementwise_blocks(n_entries, 256), 256, 0, s>>>(row_index, n_entries, n_rows,
                                                                        count, slots);
  rows_sum_kernel<<<static_cast<unsigned>(ceil_div(n_rows, 4)), 256, 0, s>>>(
      src, row_index, n_entries, n_rows, cols, count, slots, out, out_dtype);
  return check_launch("rows_sum");
}
