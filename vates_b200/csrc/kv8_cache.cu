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
  int pos_add, n, shift, dshift, align;  // log2 of the page and of dim / 16; bytes
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

// 16 bf16 values: one 32-byte access where the address allows it.
__device__ __forceinline__ void load16(uint32_t (&x)[8], const uint16_t *q, int align) {
  if (align >= 32) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]),
                   "=r"(x[6]), "=r"(x[7])
                 : "l"(q));
  } else if (align >= 16) {
    const uint4 a = ldg_v4(q), b = ldg_v4(q + 8);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = q[2 * j] | ((uint32_t)q[2 * j + 1] << 16);
  }
}
__device__ __forceinline__ void store16(uint16_t *q, const uint32_t (&x)[8], int align) {
  if (align >= 32) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(q), "r"(x[0]),
                 "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(q)[0] = make_uint4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<uint4 *>(q)[1] = make_uint4(x[4], x[5], x[6], x[7]);
  }
}

// One CTA per (page window, K or V of one head, sequence): the window's new
// rows stay in registers between the maximum and the codes, so each is read
// once. NV vectors of 16 elements per thread cover page * dim <= NV * 4096.
// HBM-bound (2 bytes read and 1 written per element: 2 x 65,536 rows of 2 heads of
// 256 take 60 us, 6.7 TB/s, a copy's rate); 16 elements per thread and 32-byte loads
// keep it from being instruction-bound. A step's few rows cost the launch, 3 us.
template <int NV>
__global__ void __launch_bounds__(KW_THREADS) kv8_append_kernel(Kv8AppendParams p) {
  __shared__ uint32_t s_max[KW_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, b = blockIdx.z;
  const int kv = blockIdx.y & 1, h = blockIdx.y >> 1;
  const int page = p.c.page;
  const int pos = p.pos[b] + p.pos_add;
  const int rows = kv8_rows(p.counts, b, p.n, blockIdx.x == 0 && tid == 0 ? p.status : nullptr);
  if (pos < 0) {
    if (rows && tid == 0) flag_status(p.status, VB_STATUS_BOUNDS);
    return;
  }
  const int idx = (pos >> p.shift) + blockIdx.x;         // page of the sequence
  const long long first = (long long)idx << p.shift;     // its first position
  if (rows == 0 || first >= (long long)pos + rows) return;
  const int lo = max(0, (int)(pos - first));                            // new rows of the page:
  const int hi = (int)min((long long)page, (long long)pos + rows - first);  // [lo, hi)
  // thread's row r0 + i step of the page, elements col .. col + 15
  const int r0 = tid >> p.dshift, col = (tid & ((1 << p.dshift) - 1)) * 16;
  const int step = KW_THREADS >> p.dshift;
  const int64_t row_step = kv ? p.st[1] : p.st[0];
  const uint16_t *src = (kv ? p.src[1] + b * p.sb[1] + h * p.sh[1]
                            : p.src[0] + b * p.sb[0] + h * p.sh[0]) +
                        (first - pos + r0) * row_step + col;
  uint32_t x[NV][8];
  uint32_t mx = 0;  // max |x| as bf16 bits, two halves
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i][j] = 0;
    const int r = r0 + i * step;
    if (r >= lo && r < hi) load16(x[i], src + i * step * row_step, p.align);
  }
  const int id = kv8_page(p.c.page_table + (size_t)b * p.c.max_pages, p.c.max_pages, p.c.pages,
                          idx, tid == 0 ? p.status : nullptr);
  if (id < 0) return;
  const size_t ph = (size_t)id * p.c.kv_heads + h;
  float *scale_p = (kv ? p.c.v_scales : p.c.k_scales) + ph;
  uint4 *codes = reinterpret_cast<uint4 *>((kv ? p.c.v_codes : p.c.k_codes) +
                                           ph * (size_t)(page * p.c.dim)) + tid;
  const float s0 = lo > 0 ? *scale_p : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = __vmaxu2(mx, x[i][j] & 0x7FFF7FFFu);
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
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = x[i][j] & 0x7FFFu, c = (x[i][j] >> 16) & 0x7FFFu;
        m = max(m, max(a < 0x7F80u ? a : 0u, c < 0x7F80u ? c : 0u));
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
    const int r = r0 + i * step;
    uint4 *dst = codes + i * KW_THREADS;
    uint32_t c[16];
    if (r >= lo && r < hi) {
      if (finite) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          c[2 * j] = rint_bits(__fmul_rn(__uint_as_float(x[i][j] << 16), inv));
          c[2 * j + 1] = rint_bits(__fmul_rn(__uint_as_float(x[i][j] & 0xFFFF0000u), inv));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          c[2 * j] = code_any(__uint_as_float(x[i][j] << 16), inv);
          c[2 * j + 1] = code_any(__uint_as_float(x[i][j] & 0xFFFF0000u), inv);
        }
      }
    } else if (grown && r < lo) {
      const uint4 o = *dst;
      const uint32_t w[4] = {o.x ^ 0x80808080u, o.y ^ 0x80808080u, o.z ^ 0x80808080u,
                             o.w ^ 0x80808080u};
#pragma unroll
      for (int j = 0; j < 16; ++j)
        c[j] = rint_bits(__fmul_rn(code_f32(w[j >> 2], j & 3), ratio));
    } else {
      continue;
    }
    *dst = make_uint4(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]),
                      pack4(c[8], c[9], c[10], c[11]), pack4(c[12], c[13], c[14], c[15]));
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
  int n, shift, dshift, align;
};

// A thread turns 16 codes into 16 bf16 values (16 bytes in, 32 out), KR_UNROLL
// times; rows past the length are written as zeros. HBM-bound: 131,072 rows of 2
// heads of 256 take 71 us, 5.7 TB/s or 0.88 of a copy.
__global__ void __launch_bounds__(KR_THREADS) kv8_read_kernel(Kv8ReadParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.z, kv = blockIdx.y & 1, h = blockIdx.y >> 1;
  const int start = p.start ? p.start[b] : 0, len = p.lens[b];
  if (start < 0 && threadIdx.x == 0) flag_status(p.status, VB_STATUS_BOUNDS);
  const int total = p.n << p.dshift;  // (n <= 2^26)
  const float *scales = (kv ? p.c.v_scales : p.c.k_scales) + h;
  const int8_t *codes = (kv ? p.c.v_codes : p.c.k_codes) + (size_t)h * p.c.page * p.c.dim;
  const uint32_t pool_step = (uint32_t)(p.c.kv_heads * p.c.page * p.c.dim);
  uint16_t *dst = (kv ? p.dst[1] : p.dst[0]) +
                  ((size_t)b * p.c.kv_heads + h) * ((size_t)p.n * p.c.dim);
  const int base = blockIdx.x * (KR_THREADS * KR_UNROLL) + threadIdx.x;
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
  int id[KR_UNROLL];
#pragma unroll
  for (int i = 0; i < KR_UNROLL; ++i) {
    const int v = base + i * KR_THREADS;
    const long long at = (long long)start + (v >> p.dshift);
    id[i] = v < total && at >= 0 && at < len
                ? kv8_page(table, p.c.max_pages, p.c.pages, (int)(at >> p.shift), p.status) : -1;
  }
  uint4 w[KR_UNROLL];
  float s[KR_UNROLL];
#pragma unroll
  for (int i = 0; i < KR_UNROLL; ++i) {
    w[i] = make_uint4(0, 0, 0, 0);
    s[i] = 0.f;
    if (id[i] >= 0) {
      const int v = base + i * KR_THREADS;
      const int r = (start + (v >> p.dshift)) & (p.c.page - 1);
      s[i] = __ldg(scales + (size_t)id[i] * p.c.kv_heads);
      w[i] = ldg_nc_v4(codes + (size_t)id[i] * pool_step + r * p.c.dim +
                       (v & ((1 << p.dshift) - 1)) * 16);
    }
  }
#pragma unroll
  for (int i = 0; i < KR_UNROLL; ++i) {
    const int v = base + i * KR_THREADS;
    if (v >= total) continue;
    const uint32_t u[4] = {w[i].x ^ 0x80808080u, w[i].y ^ 0x80808080u, w[i].z ^ 0x80808080u,
                           w[i].w ^ 0x80808080u};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = pack_bf2(__fmul_rn(code_f32(u[j >> 1], 2 * (j & 1)), s[i]),
                      __fmul_rn(code_f32(u[j >> 1], 2 * (j & 1) + 1), s[i]));
    store16(dst + (size_t)v * 16, o, p.align);
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
  int64_t odd = 0;  // low bits of every row's offset in elements
  for (int i = 0; i < 2; ++i) {
    const int64_t *st = i ? a->v_strides : a->k_strides;
    p.sb[i] = st[0]; p.sh[i] = st[1]; p.st[i] = st[2];
    odd |= (int64_t)((uintptr_t)p.src[i] / 2) | st[0] | st[1] | st[2];
    VB_REQUIRE((uintptr_t)p.src[i] % 2 == 0, "vb_kv8_append: odd address");
  }
  p.pos = a->pos; p.counts = a->counts; p.status = a->status;
  p.pos_add = a->pos_add; p.n = a->n;
  p.align = odd % 16 == 0 ? 32 : odd % 8 == 0 ? 16 : 2;
  p.shift = kv8_page_shift(p.c.page);
  p.dshift = p.c.dim == 64 ? 2 : p.c.dim == 128 ? 3 : 4;
  const int windows = (int)(((long long)a->n + p.c.page - 2) / p.c.page) + 1;
  const dim3 grid(windows, p.c.kv_heads * 2, p.c.batch), block(KW_THREADS);
  cudaStream_t s = as_stream(stream);
  switch (p.c.page * p.c.dim / (16 * KW_THREADS)) {
    case 0: case 1: vb_launch(kv8_append_kernel<1>, grid, block, 0, s, true, p); break;
    case 2: vb_launch(kv8_append_kernel<2>, grid, block, 0, s, true, p); break;
    case 4: vb_launch(kv8_append_kernel<4>, grid, block, 0, s, true, p); break;
    default: vb_launch(kv8_append_kernel<8>, grid, block, 0, s, true, p); break;
  }
  return check_launch("kv8_append_kernel");
}

int vb_kv8_read(const VbKv8ReadArgs *a, vb_stream_t stream) {
  VB_REQUIRE(a, "vb_kv8_read: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_read");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->n >= 0 && a->n <= 1 << 26, "vb_kv8_read: n=%d (<= 2^26)", a->n);
  if (a->n == 0) return VB_OK;
  VB_REQUIRE(a->lens && a->keys && a->values, "vb_kv8_read: null tensor");
  VB_REQUIRE(((uintptr_t)a->keys % 16) == 0 && ((uintptr_t)a->values % 16) == 0,
             "vb_kv8_read: outputs must be 16-byte aligned");
  Kv8ReadParams p;
  p.c = a->cache;
  p.lens = a->lens; p.start = a->start;
  p.dst[0] = a->keys; p.dst[1] = a->values;
  p.status = a->status; p.n = a->n;
  p.align = ((uintptr_t)a->keys % 32) || ((uintptr_t)a->values % 32) ? 16 : 32;
  p.shift = kv8_page_shift(p.c.page);
  p.dshift = p.c.dim == 64 ? 2 : p.c.dim == 128 ? 3 : 4;
  const long long per = KR_THREADS * KR_UNROLL;
  const long long blocks = ((long long)a->n * (p.c.dim / 16) + per - 1) / per;
  vb_launch(kv8_read_kernel, dim3((unsigned)blocks, p.c.kv_heads * 2, p.c.batch),
            dim3(KR_THREADS), 0, as_stream(stream), true, p);
  return check_launch("kv8_read_kernel");
}

}  // extern "C"
