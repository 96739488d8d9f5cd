// Attention weight that the rows of the paged 8-bit cache receive, added up:
//
//   w_j += sum over query heads of the kv head, rows i that see j, of
//          exp(scale * q_i . k_j - lse_i)
//
// with lse_i from the attention itself, so no row needs another key than j and
// V is not read. The products are those of the attention kernels: codes and
// queries (after a power of two per row) are exact in f16, sums float32.
//
// A warp takes 16 keys at a time straight from global memory into the fragments
// of the product S^T = K q^T (lane (g, c) has 16 consecutive bytes of keys g and
// g + 8, four k-steps), and all query rows of the kv head in turn, 8 to a
// fragment, from shared memory. A key's weights are added up in the lane, then
// over the four lanes that have the key: one order, whatever the launch.
#include "kv8_attn.cuh"

namespace vb {
namespace {

constexpr int WG_THREADS = 128;
constexpr int WG_ROWS = 32;  // query rows in shared memory at a time

struct Kv8WeighParams {
  Kv8AttnParams a;           // out, lse (written) and workspace are not used
  const float *lse;
  const int32_t *fresh, *seen;  // new rows at the end (null: the query rows), tokens so far
  float *weights;
  int32_t *positions;
  int room, groups;          // 16-key groups of a warp
};

__device__ __forceinline__ void wg_mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

template <int D>
__global__ void __launch_bounds__(WG_THREADS) kv8_weigh_kernel(const __grid_constant__ Kv8WeighParams w) {
  const Kv8AttnParams &p = w.a;
  __shared__ uint32_t s_q[WG_ROWS / 8 * D * 4];  // [8 rows][D/32][32 lanes][4]
  __shared__ float2 s_row[WG_ROWS];              // score factor, log2 sum
  __shared__ int s_vis[WG_ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int H = p.c.kv_heads, b = blockIdx.z, h = blockIdx.y;
  const bool flag = blockIdx.x == 0 && h == 0 && tid == 0;
  Kv8Span sp = kv8_span(p, b, flag);
  if (sp.keys > w.room) {
    if (flag) flag_status(p.status, VB_STATUS_BOUNDS);
    return;
  }
  const int fresh = sp.keys - (w.fresh ? kv8_rows(w.fresh, b, sp.keys, flag ? p.status : nullptr)
                                       : min(sp.q_len, sp.keys));
  const int key_first = blockIdx.x * (WG_THREADS / 32 * 16) * w.groups;
  if (key_first >= sp.keys) return;
  const int rows = sp.q_len * p.rep;
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
  const size_t at0 = ((size_t)b * H + h) * w.room;
  const size_t page_bytes = (size_t)p.c.page * D;

  for (int grp = 0; grp < w.groups; ++grp) {
    const int key0 = key_first + (grp * (WG_THREADS / 32) + warp) * 16;  // uniform in the warp
    const bool some = key0 < sp.keys;
    uint4 lo[D / 64], hi[D / 64];
    float ks = 0.f;
    if (some) {
      const int id = kv8_page(table, p.c.max_pages, p.c.pages, key0 >> p.shift,
                              lane == 0 ? p.status : nullptr);
      if (id >= 0) {
        const size_t ph = (size_t)id * H + h;
        const int8_t *k = p.c.k_codes + ph * page_bytes +
                          (size_t)((key0 & (p.c.page - 1)) + g) * D + c * 16;
        ks = __ldg(p.c.k_scales + ph);
#pragma unroll
        for (int s = 0; s < D / 64; ++s) {
          lo[s] = ldg_nc_v4(k + s * 64);
          hi[s] = ldg_nc_v4(k + s * 64 + 8 * D);
        }
      } else {
        ks = -1.f;
      }
    }
    if (ks < 0.f || !some) {
#pragma unroll
      for (int s = 0; s < D / 64; ++s) lo[s] = hi[s] = make_uint4(0, 0, 0, 0);
    }
    float sum0 = 0.f, sum1 = 0.f;  // keys g and g + 8
    for (int r0 = 0; r0 < rows; r0 += WG_ROWS) {
      if (grp == 0 || rows > WG_ROWS) {
        // ---- queries in the order of the B fragments: D / 8 lanes per row
        if (grp > 0 || r0 > 0) __syncthreads();
        constexpr int LPR = D / 8, PASS = WG_THREADS / LPR;
        const int c8 = tid % LPR;
#pragma unroll 4
        for (int k = 0; k < WG_ROWS / PASS; ++k) {
          const int r = tid / LPR + k * PASS, R = r0 + r, i = p.row_of(R), hr = R - i * p.rep;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (R < rows)
            v = kv8_load8(p.q + b * p.qb + (int64_t)(h * p.rep + hr) * p.qh + (int64_t)i * p.ql +
                              c8 * 8, p.vec);
          const float pw = kv8_q_scale<LPR>(v);
          if (c8 == 0) {
            float l = -INFINITY;
            if (R < rows) l = w.lse[((size_t)b * p.Hq + h * p.rep + hr) * p.L + i];
            const bool counts = fabsf(l) <= 3.4028235e38f;
            if (!counts && l != -INFINITY && key_first == 0 && grp == 0 && R < rows)
              flag_status(p.status, VB_STATUS_NONFINITE);
            s_row[r] = make_float2(p.scale_log2 / pw, l * 1.4426950408889634f);
            s_vis[r] = counts ? sp.visible(i) : 0;
          }
          const int fl = (r & 7) * 4 + ((c8 & 7) >> 1);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int step = (c8 >> 3) * 4 + (c8 & 1) * 2 + j;
            *reinterpret_cast<uint2 *>(
                s_q + (((r >> 3) * (D / 32) + (step >> 1)) * 32 + fl) * 4 + (step & 1) * 2) =
                j ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y);
          }
        }
        __syncthreads();
      }
      const int eights = (min(rows - r0, WG_ROWS) + 7) >> 3;
      for (int n = 0; n < eights; ++n) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D / 64; ++s) {
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const uint32_t x = (r4 == 0 ? lo[s].x : r4 == 1 ? lo[s].y : r4 == 2 ? lo[s].z : lo[s].w) ^ 0x80808080u;
            const uint32_t y = (r4 == 0 ? hi[s].x : r4 == 1 ? hi[s].y : r4 == 2 ? hi[s].z : hi[s].w) ^ 0x80808080u;
            const uint4 a = make_uint4(h2_codes(__byte_perm(x, 0x64646464u, 0x4140)),
                                       h2_codes(__byte_perm(y, 0x64646464u, 0x4140)),
                                       h2_codes(__byte_perm(x, 0x64646464u, 0x4342)),
                                       h2_codes(__byte_perm(y, 0x64646464u, 0x4342)));
            const int step = s * 4 + r4;
            const uint2 bq = *reinterpret_cast<const uint2 *>(
                s_q + ((n * (D / 32) + (step >> 1)) * 32 + lane) * 4 + (step & 1) * 2);
            wg_mma(acc, a, bq.x, bq.y);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // rows 8 n + 2 c + u
          const int r = n * 8 + 2 * c + u;
          const float2 f = s_row[r];
          const int vis = s_vis[r];
          const float z0 = fmaf(acc[u], f.x * ks, -f.y), z1 = fmaf(acc[2 + u], f.x * ks, -f.y);
          if (key0 + g < vis) sum0 += kv8_ex2(z0);
          if (key0 + g + 8 < vis) sum1 += kv8_ex2(z1);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, o);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
    }
    if (some && c < 2) {
      const int key = key0 + g + 8 * c;
      const float sum = ks < 0.f ? 0.f : c ? sum1 : sum0;
      if (key < sp.keys) {
        const bool is_new = key >= fresh;
        if (is_new || sum != 0.f) w.weights[at0 + key] = (is_new ? 0.f : w.weights[at0 + key]) + sum;
        if (is_new && w.positions) w.positions[at0 + key] = w.seen[b] - (sp.keys - key);
      }
    }
  }
}

template <int D>
int wg_run(Kv8WeighParams &w, cudaStream_t s) {
  const VbKv8Cache &c = w.a.c;
  const long long cap = (long long)c.max_pages * c.page;
  const long long keys = cap < w.room ? cap : w.room, per = WG_THREADS / 32 * 16;
  const long long units = (long long)c.batch * c.kv_heads;
  // keys of a CTA: a few groups a warp once that still fills the SMs
  w.groups = 1;
  while (w.groups < 4 && (keys + per * w.groups - 1) / (per * w.groups) * units > 148 * 16)
    w.groups *= 2;
  const long long blocks = (keys + per * w.groups - 1) / (per * w.groups);
  if (blocks == 0) return VB_OK;
  vb_launch(kv8_weigh_kernel<D>, dim3((unsigned)blocks, c.kv_heads, c.batch), dim3(WG_THREADS), 0, s,
            true, w);
  return check_launch("kv8_weigh_kernel");
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_kv8_weigh(const VbKv8WeighArgs *a, vb_stream_t stream) {
  VB_REQUIRE(a, "vb_kv8_weigh: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_weigh");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->q_heads >= 1 && a->q_heads % a->cache.kv_heads == 0 &&
                 a->q_heads / a->cache.kv_heads <= 128,
             "vb_kv8_weigh: %d query heads over %d kv heads (at most 128 each)", a->q_heads,
             a->cache.kv_heads);
  VB_REQUIRE(a->L >= 0 && (long long)a->L * a->q_heads <= 1 << 24,
             "vb_kv8_weigh: L=%d rows of %d heads", a->L, a->q_heads);
  VB_REQUIRE(a->room >= 0 && a->room <= 0x7fffffff - 65536, "vb_kv8_weigh: room=%d", a->room);
  VB_REQUIRE(a->lens && (a->L == 0 || (a->q && a->lse)) && (a->weights || a->room == 0),
             "vb_kv8_weigh: null tensor");
  VB_REQUIRE(!a->positions || a->seen, "vb_kv8_weigh: positions without seen");
  VB_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "vb_kv8_weigh: scale %g", (double)a->scale);
  VB_REQUIRE(a->cache.kv_heads <= 65535, "vb_kv8_weigh: too many heads");
  Kv8WeighParams w = {};
  Kv8AttnParams &p = w.a;
  p.c = a->cache;
  p.q = a->q;
  p.qb = a->q_strides[0]; p.qh = a->q_strides[1]; p.ql = a->q_strides[2];
  p.lens = a->lens; p.q_lens = a->q_lens; p.status = a->status;
  p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
  p.Hq = a->q_heads; p.L = a->L; p.rep = a->q_heads / a->cache.kv_heads;
  p.len_add = a->len_add; p.causal = a->causal ? 1 : 0;
  p.shift = kv8_page_shift(a->cache.page);
  p.vec = ((uintptr_t)a->q % 16) == 0 && p.qb % 8 == 0 && p.qh % 8 == 0 && p.ql % 8 == 0;
  p.rep_inv = (uint32_t)((1ull << 32) / (uint32_t)p.rep) + (p.rep > 1);
  w.lse = a->lse; w.fresh = a->fresh; w.seen = a->seen;
  w.weights = a->weights; w.positions = a->positions; w.room = a->room;
  cudaStream_t s = as_stream(stream);
  switch (a->cache.dim) {
    case 64: return wg_run<64>(w, s);
    case 128: return wg_run<128>(w, s);
    default: return wg_run<256>(w, s);
  }
}
