// The host's side of the products over rows: the checks that every entry point makes of
// its list and sizes, and products of few rows (linear_few.hip: forward only, any
// alignment).
#pragma once

#include "linear_tile.h"

namespace mgq {

// The low bits of where the operands' rows start and end (n bytes each).
inline uintptr_t lin_row_bounds(const LinArgs& a, int64_t n) {
  return reinterpret_cast<uintptr_t>(a.P) | reinterpret_cast<uintptr_t>(a.Q) |
         static_cast<uintptr_t>(a.ldp | a.ldq | a.p_group | n);
}
// A workgroup computes 16 nq entries (nq = 1, 2 or 4) by lin_few_cols(nq) weight rows.
inline int lin_few_cols(int nq) { return nq == 4 ? 32 : 16; }
inline int64_t lin_few_grid(const LinArgs& a, int nq) {
  return lin_row_tiles(a, 16 * nq) * ceil_div(a.np, lin_few_cols(nq));
}
constexpr int64_t kLinFewGrid = int64_t(1) << 24;  // 256 threads each, less than 2^32 in all
int lin_few_rows(const LinArgs& a, int op, int nq, hipStream_t s, const char* what);

inline int lin_check_list(const char* what, const int32_t* offsets, const int32_t* row_index,
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

inline int lin_check_dims(const char* what, int64_t N, int64_t K) {
  MGQ_REQUIRE(N >= 1 && K >= 0 && N < (int64_t(1) << 30) && K < (int64_t(1) << 30), MGQ_ERR_SHAPE,
              "%s: bad weight shape [%lld, %lld]", what, (long long)N, (long long)K);
  return MGQ_OK;
}

}  // namespace mgq
