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

// 0x4B400000 + c as a float is 1.5 * 2^23 + c: adding 1.5 * 2^23 rounds to the
// nearest integer (ties to even) and leaves its two's complement in the low
// byte; exact for |v| <= 2^21.
__device__ __forceinline__ uint32_t rint_bits(float v) {
  return __float_as_uint(__fadd_rn(v, 12582912.f));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Byte j of a word of codes + 128 as float: 2^23 + u is exact, and so is the
// difference.
__device__ __forceinline__ float code_f32(uint32_t u, int j) {
  return __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + j)) - 8388736.f;
}
// 16 codes under another scale: rint(code * (old / new)), as the append kernel
// rewrites a page that grows.
__device__ __forceinline__ uint4 kv8_recode(const uint4 &o, float ratio) {
  const uint32_t w[4] = {o.x ^ 0x80808080u, o.y ^ 0x80808080u, o.z ^ 0x80808080u,
                         o.w ^ 0x80808080u};
  uint32_t c[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) c[j] = rint_bits(__fmul_rn(code_f32(w[j >> 2], j & 3), ratio));
  return make_uint4(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]),
                    pack4(c[8], c[9], c[10], c[11]), pack4(c[12], c[13], c[14], c[15]));
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
