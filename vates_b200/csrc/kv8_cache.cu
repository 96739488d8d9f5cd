// Writing and reading the paged 8-bit KV cache.
//
// Every (page, kv head) of K and of V has one float32 scale s; a stored value
// is code * s with an int8 code in [-127, 127]. Writing rows x into a page
// that already holds older rows under scale s0 (s0 = 0 for an empty page):
//   s = max(s0, max(max|x| / 127, 2^-40))      (s0 while max|x| = 0)
//   code(x) = rint(x * (1 / s)),  older code -> rint(code * (s0 / s))
// so a page's scale only grows while it fills, and the older rows are
// rewritten only when it does. All of it in float32, each product rounded
// once, ties to even. An infinity takes the code +-127 and a NaN 0 (neither
// enters the maximum); both raise VB_STATUS_NONFINITE.
#include "kv8.cuh"

namespace vb {
namespace {

constexpr int KW_THREADS = 256;

struct Kv8AppendParams {
  VbKv8Cache c;
  const uint16_t *src[2];
  int64_t sb[2], sh[2], st[2];  // element strides of batch, head, row
  const int32_t *pos, *counts;
  int32_t *status;
  int pos_add, n, shift, dshift, vec;  // log2 of the page and of dim / 8
};

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
// Code of one value, any bits.
__device__ __forceinline__ uint32_t code_any(float x, float inv) {
  const float v = x == x && inv > 0.f ? fminf(fmaxf(__fmul_rn(x, inv), -127.f), 127.f) : 0.f;
  return rint_bits(v);
}

// One CTA per (page window, K or V of one head, sequence): the window's new
// rows stay in registers between the maximum and the codes, so each is read
// once. NV 8-element vectors per thread cover page * dim <= NV * 2048.
template <int NV>
__global__ void __launch_bounds__(KW_THREADS) kv8_append_kernel(Kv8AppendParams p) {
  __shared__ uint32_t s_max[KW_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, b = blockIdx.z;
  const int kv = blockIdx.y & 1, h = blockIdx.y >> 1;
  const int page = p.c.page, dim = p.c.dim;
  const int pos = p.pos[b] + p.pos_add;
  const int rows = kv8_rows(p.counts, b, p.n, blockIdx.x == 0 && tid == 0 ? p.status : nullptr);
  if (pos < 0) {
    if (rows && tid == 0) flag_status(p.status, VB_STATUS_BOUNDS);
    return;
  }
  const int idx = (pos >> p.shift) + blockIdx.x;         // page of the sequence
  const long long first = (long long)idx << p.shift;     // its first position
  if (rows == 0 || first >= (long long)pos + rows) return;
  const int id = kv8_page(p.c.page_table + (size_t)b * p.c.max_pages, p.c.max_pages, p.c.pages,
                          idx, tid == 0 ? p.status : nullptr);
  if (id < 0) return;
  const int lo = max(0, (int)(pos - first));                            // new rows of the page:
  const int hi = (int)min((long long)page, (long long)pos + rows - first);  // [lo, hi)
  const size_t ph = (size_t)id * p.c.kv_heads + h;
  float *scale_p = (kv ? p.c.v_scales : p.c.k_scales) + ph;
  int8_t *codes = (kv ? p.c.v_codes : p.c.k_codes) + ph * (size_t)(page * dim);
  const float s0 = lo > 0 ? *scale_p : 0.f;
  const uint16_t *src = kv ? p.src[1] + b * p.sb[1] + h * p.sh[1]
                           : p.src[0] + b * p.sb[0] + h * p.sh[0];
  const int64_t row_step = kv ? p.st[1] : p.st[0];
  const int row0 = (int)(first - pos);                   // source row of page row 0

  uint4 x[NV];
  uint32_t mx = 0;                                        // max |x| as bf16 bits, two halves
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tid + i * KW_THREADS, r = v >> p.dshift;
    const int col = (v & ((1 << p.dshift) - 1)) * 8;
    x[i] = make_uint4(0, 0, 0, 0);
    if (r >= lo && r < hi) {
      const uint16_t *q = src + (int64_t)(row0 + r) * row_step + col;
      if (p.vec) {
        x[i] = ldg_nc_v4(q);
      } else {
        x[i].x = q[0] | ((uint32_t)q[1] << 16);
        x[i].y = q[2] | ((uint32_t)q[3] << 16);
        x[i].z = q[4] | ((uint32_t)q[5] << 16);
        x[i].w = q[6] | ((uint32_t)q[7] << 16);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    constexpr uint32_t A = 0x7FFF7FFFu;
    mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(x[i].x & A, x[i].y & A), __vmaxu2(x[i].z & A, x[i].w & A)));
  }
  uint32_t m = max(mx & 0xFFFFu, mx >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) s_max[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KW_THREADS / 32; ++w) m = max(m, s_max[w]);
  const bool finite = m < 0x7F80u;
  if (!finite) {  // (rare) the maximum over the finite values alone
    if (tid == 0) flag_status(p.status, VB_STATUS_NONFINITE);
    m = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = u[j] & 0x7FFFu, c = (u[j] >> 16) & 0x7FFFu;
        m = max(m, max(a < 0x7F80u ? a : 0u, c < 0x7F80u ? c : 0u));
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    __syncthreads();
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KW_THREADS / 32; ++w) m = max(m, s_max[w]);
  }
  const float amax = bf2f((uint16_t)m);
  const float s = fmaxf(s0, amax > 0.f ? fmaxf(__fdiv_rn(amax, 127.f), KV8_MIN_SCALE) : 0.f);
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
  if (tid == 0) *scale_p = s;
  const bool grown = lo > 0 && s > s0;
  const float ratio = grown ? __fdiv_rn(s0, s) : 1.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = tid + i * KW_THREADS, r = v >> p.dshift;
    uint2 *dst = reinterpret_cast<uint2 *>(codes) + v;
    if (r >= lo && r < hi) {
      const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t c[8];
      if (finite) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[2 * j] = rint_bits(__fmul_rn(__uint_as_float(u[j] << 16), inv));
          c[2 * j + 1] = rint_bits(__fmul_rn(__uint_as_float(u[j] & 0xFFFF0000u), inv));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[2 * j] = code_any(__uint_as_float(u[j] << 16), inv);
          c[2 * j + 1] = code_any(__uint_as_float(u[j] & 0xFFFF0000u), inv);
        }
      }
      *dst = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
    } else if (grown && r < lo) {
      const uint2 o = *dst;
      uint32_t c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = j < 4 ? o.x : o.y;
        c[j] = rint_bits(__fmul_rn(code_f32(w ^ 0x80808080u, j & 3), ratio));
      }
      *dst = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
    }
  }
}

// ----------------------------------------------------------------- read back
constexpr int KR_THREADS = 256;
constexpr int KR_UNROLL = 4;

struct Kv8ReadParams {
  VbKv8Cache c;
  const int32_t *lens, *start;
  uint16_t *dst[2];
  int32_t *status;
  int n, shift, dshift;
};

// One thread turns 8 codes into 8 bf16 values (8 bytes in, 16 out), KR_UNROLL
// times; rows past the sequence's length are written as zeros.
__global__ void __launch_bounds__(KR_THREADS) kv8_read_kernel(Kv8ReadParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.z, kv = blockIdx.y & 1, h = blockIdx.y >> 1;
  const int dim = p.c.dim;
  const int start = p.start ? p.start[b] : 0, len = p.lens[b];
  if (start < 0 && threadIdx.x == 0) flag_status(p.status, VB_STATUS_BOUNDS);
  const long long total = (long long)p.n << p.dshift;
  const float *scales = kv ? p.c.v_scales : p.c.k_scales;
  const int8_t *codes = kv ? p.c.v_codes : p.c.k_codes;
  uint4 *dst = reinterpret_cast<uint4 *>(kv ? p.dst[1] : p.dst[0]) +
              ((long long)b * p.c.kv_heads + h) * total;
  const long long base = (long long)blockIdx.x * (KR_THREADS * KR_UNROLL) + threadIdx.x;
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
  uint2 w[KR_UNROLL];
  float s[KR_UNROLL];
#pragma unroll
  for (int i = 0; i < KR_UNROLL; ++i) {
    const long long v = base + i * KR_THREADS;
    w[i] = make_uint2(0, 0);
    s[i] = 0.f;
    if (v < total) {
      const long long at = start + (v >> p.dshift);
      if (at >= 0 && at < len) {
        const int id = kv8_page(table, p.c.max_pages, p.c.pages, (int)(at >> p.shift), p.status);
        if (id >= 0) {
          const size_t ph = (size_t)id * p.c.kv_heads + h;
          s[i] = __ldg(scales + ph);
          w[i] = ldg_nc_v2(codes + (ph * p.c.page + (at & (p.c.page - 1))) * dim +
                           (int)(v & ((1 << p.dshift) - 1)) * 8);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < KR_UNROLL; ++i) {
    const long long v = base + i * KR_THREADS;
    if (v >= total) continue;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[j] = __fmul_rn(code_f32((j < 4 ? w[i].x : w[i].y) ^ 0x80808080u, j & 3), s[i]);
    dst[v] = make_uint4(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]),
                        pack_bf2(f[6], f[7]));
  }
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

int vb_kv8_append(const VbKv8AppendArgs *a, vb_stream_t stream) {
  VB_REQUIRE(a, "vb_kv8_append: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_append");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->n >= 0, "vb_kv8_append: n=%d", a->n);
  if (a->n == 0) return VB_OK;
  VB_REQUIRE(a->keys && a->values && a->pos, "vb_kv8_append: null tensor");
  Kv8AppendParams p;
  p.c = a->cache;
  p.src[0] = a->keys; p.src[1] = a->values;
  int vec = 1;
  for (int i = 0; i < 2; ++i) {
    const int64_t *st = i ? a->v_strides : a->k_strides;
    p.sb[i] = st[0]; p.sh[i] = st[1]; p.st[i] = st[2];
    if (((uintptr_t)p.src[i] % 16) || st[0] % 8 || st[1] % 8 || st[2] % 8) vec = 0;
  }
  p.pos = a->pos; p.counts = a->counts; p.status = a->status;
  p.pos_add = a->pos_add; p.n = a->n; p.vec = vec;
  p.shift = kv8_page_shift(p.c.page);
  p.dshift = p.c.dim == 64 ? 3 : p.c.dim == 128 ? 4 : 5;
  const int windows = (int)(((long long)a->n + p.c.page - 2) / p.c.page) + 1;
  const dim3 grid(windows, p.c.kv_heads * 2, p.c.batch), block(KW_THREADS);
  cudaStream_t s = as_stream(stream);
  switch (p.c.page * p.c.dim / (8 * KW_THREADS)) {
    case 0: case 1: vb_launch(kv8_append_kernel<1>, grid, block, 0, s, false, p); break;
    case 2: vb_launch(kv8_append_kernel<2>, grid, block, 0, s, false, p); break;
    case 4: vb_launch(kv8_append_kernel<4>, grid, block, 0, s, false, p); break;
    case 8: vb_launch(kv8_append_kernel<8>, grid, block, 0, s, false, p); break;
    default: vb_launch(kv8_append_kernel<16>, grid, block, 0, s, false, p); break;
  }
  return check_launch("kv8_append_kernel");
}

int vb_kv8_read(const VbKv8ReadArgs *a, vb_stream_t stream) {
  VB_REQUIRE(a, "vb_kv8_read: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_read");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->n >= 0, "vb_kv8_read: n=%d", a->n);
  if (a->n == 0) return VB_OK;
  VB_REQUIRE(a->lens && a->keys && a->values, "vb_kv8_read: null tensor");
  VB_REQUIRE(((uintptr_t)a->keys % 16) == 0 && ((uintptr_t)a->values % 16) == 0,
             "vb_kv8_read: outputs must be 16-byte aligned");
  Kv8ReadParams p;
  p.c = a->cache;
  p.lens = a->lens; p.start = a->start;
  p.dst[0] = a->keys; p.dst[1] = a->values;
  p.status = a->status; p.n = a->n;
  p.shift = kv8_page_shift(p.c.page);
  p.dshift = p.c.dim == 64 ? 3 : p.c.dim == 128 ? 4 : 5;
  const long long per = KR_THREADS * KR_UNROLL;
  const long long blocks = ((long long)a->n * (p.c.dim / 8) + per - 1) / per;
  vb_launch(kv8_read_kernel, dim3((unsigned)blocks, p.c.kv_heads * 2, p.c.batch),
            dim3(KR_THREADS), 0, as_stream(stream), false, p);
  return check_launch("kv8_read_kernel");
}

}  // extern "C"
