// Paged 8-bit KV cache: device view and host-side checks shared by the
// kernels that write, read and attend it.
#pragma once

#include "common.cuh"

namespace vb {

// Smallest scale of a page that holds a non-zero value: keeps 1 / scale and
// the ratio of two scales finite in float32 (values below 2^-41 read as 0).
constexpr float KV8_MIN_SCALE = 9.094947017729282e-13f;  // 2^-40

// Entry `idx` of a sequence's page table (-1 past its end). Looking at the value
// is left to kv8_page_ok, so that a prefetch does not wait for the load.
__device__ __forceinline__ int kv8_page_load(const int32_t *table, int max_pages, int idx) {
  return idx >= 0 && idx < max_pages ? __ldg(table + idx) : -1;
}
// The pool page, or -1 (flagged) when the table is too short or names a page
// outside the pool.
__device__ __forceinline__ int kv8_page_ok(int id, int pages, int32_t *status) {
  if ((unsigned)id < (unsigned)pages) return id;
  flag_status(status, VB_STATUS_BOUNDS);
  return -1;
}
__device__ __forceinline__ int kv8_page(const int32_t *table, int max_pages, int pages, int idx,
                                        int32_t *status) {
  return kv8_page_ok(kv8_page_load(table, max_pages, idx), pages, status);
}

// Rows of one sequence in this call: counts[b] clipped to [0, n], or n.
__device__ __forceinline__ int kv8_rows(const int32_t *counts, int b, int n, int32_t *status) {
  if (!counts) return n;
  const int c = counts[b];
  if (c < 0 || c > n) flag_status(status, VB_STATUS_BOUNDS);
  return min(max(c, 0), n);
}

// log2 of a page size (16, 32, 64 or 128), or -1.
static inline int kv8_page_shift(int page) {
  return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1;
}

static inline int kv8_check(const VbKv8Cache *c, const char *what) {
  VB_REQUIRE(c, "%s: null cache", what);
  VB_REQUIRE(c->dim == 64 || c->dim == 128 || c->dim == 256,
             "%s: head dim %d (64, 128 or 256)", what, c->dim);
  VB_REQUIRE(kv8_page_shift(c->page) >= 0, "%s: page of %d rows (16, 32, 64 or 128)", what,
             c->page);
  VB_REQUIRE(c->pages >= 1 && c->kv_heads >= 1 && c->kv_heads <= 16384 && c->batch >= 1 &&
                 c->batch <= 65535 && c->max_pages >= 1,
             "%s: pages=%d kv_heads=%d (<= 16384) batch=%d (<= 65535) max_pages=%d", what,
             c->pages, c->kv_heads, c->batch, c->max_pages);
  VB_REQUIRE((long long)c->max_pages * c->page <= 0x7fffffffll - 65536,
             "%s: %d pages of %d rows exceed 31-bit positions", what, c->max_pages, c->page);
  VB_REQUIRE(c->k_codes && c->v_codes && c->k_scales && c->v_scales && c->page_table,
             "%s: null cache tensor", what);
  VB_REQUIRE(((uintptr_t)c->k_codes % 16) == 0 && ((uintptr_t)c->v_codes % 16) == 0,
             "%s: codes must be 16-byte aligned", what);
  return VB_OK;
}

}  // namespace vb
