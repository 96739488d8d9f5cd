// Attention over the paged 8-bit KV cache, few query rows per kv head (decode
// and verify steps): HBM-bound, one byte per cached value.
//
//   z = scale * s_K(page) * (q . code_K),  o = sum_j 2^(z_j log2 e - m) s_V(page_j) code_V / l
//
// The codes are exact in f16 and so are the queries after a power of two per
// row, so q . code runs on f16 tensor-core products with float32 sums; the
// scales are applied to the sums. The weights are rounded to f16 (11 bits)
// after a factor s_V(page) / v, v the largest V scale so far; l is summed in
// float32 from the unrounded weights.
//
// A CTA (8 warps) owns up to 32 query rows of one kv head and a range of keys,
// in tiles of 16 KB of K and of V that cp.async brings into a ring (the rows
// of a page are contiguous; chunks of 16 bytes are XOR-swizzled so that both
// fragment reads below are free of bank conflicts):
//   S: warp w takes 2048 / D keys of the tile over all of D; lane (g, c) of an
//      8-key group reads 16 consecutive bytes of key g, four k-steps of the
//      product (the order of dims within a 64-dim span is the same permutation
//      for q);
//   max over the warps through shared memory, weights as PV's A fragments;
//   PV: warp takes 32 dims and four 16-key steps; lane (g, c) reads 4 bytes of
//      its four keys and interleaves them into key pairs.
// Key ranges ("splits") of one row tile meet in kv8_combine_kernel.
#include "kv8_attn.cuh"

namespace vb {
namespace {

constexpr int KA_THREADS = 256;
constexpr int KA_TILE = 16384;  // bytes of K, and of V, per tile

template <int D, int MT>
struct Kv8Tile {
  static constexpr int KT = KA_TILE / D;            // keys per tile
  static constexpr int NTW = KT / 64;               // 8-key groups per warp
  static constexpr int NKG = KT / 64;               // key groups of PV (32-dim groups: 8 / NKG)
  static constexpr int STAGES = MT == 1 ? 3 : 2;
  static constexpr int MAXP = KT / 16;              // most pages per tile
  static constexpr int Q_BYTES = MT * D / 16 * 512;
  static constexpr int P_BYTES = MT * KT / 16 * 512;
  static constexpr int RING = STAGES * 2 * KA_TILE;
  static constexpr int SMEM = RING + Q_BYTES + P_BYTES;
};

// Byte offset of 16-byte chunk ch of a key in a tile.
template <int D>
__device__ __forceinline__ uint32_t ka_chunk(int key, int ch) {
  if (D == 64)
    return (uint32_t)((key >> 1) * 128 +
                      (((((key & 1) << 2) | ch) ^ (((key >> 1) & 3) << 1)) << 4));
  return (uint32_t)(key * D + ((ch ^ (((key >> 1) & 3) << 1) ^ ((key & 1) << 2)) << 4));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

template <int D, int MT>
__global__ void __launch_bounds__(KA_THREADS, 2) kv8_attn_kernel(Kv8AttnParams p) {
  using T = Kv8Tile<D, MT>;
  constexpr int KT = T::KT, ROWS = 16 * MT;
  extern __shared__ __align__(128) uint8_t smem[];
  uint4 *s_q = reinterpret_cast<uint4 *>(smem + T::RING);                // [MT][D/16][32]
  uint32_t *s_p = reinterpret_cast<uint32_t *>(smem + T::RING + T::Q_BYTES);  // [MT][KT/16][32][4]
  __shared__ float s_ks[T::STAGES][T::MAXP], s_vs[T::STAGES][T::MAXP];
  __shared__ __align__(16) float s_max[ROWS][8];
  __shared__ float s_fac[ROWS], s_l[8][ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const int split = blockIdx.x, b = blockIdx.z;
  const int h = blockIdx.y / p.row_tiles, rt = blockIdx.y % p.row_tiles;
  const int r_base = rt * ROWS, rows = p.L * p.rep;
  const Kv8Span sp = kv8_span(p, b, split == 0 && blockIdx.y == 0 && tid == 0);
  const int i_last = min(min(r_base + ROWS, rows) - 1, sp.q_len * p.rep - 1) / p.rep;
  const int kend = r_base < sp.q_len * p.rep ? sp.visible(i_last) : 0;
  const int tiles = (kend + KT - 1) / KT;
  const int t0 = (int)((long long)tiles * split / p.splits);
  const int t1 = (int)((long long)tiles * (split + 1) / p.splits);
  const size_t tile_id = (((size_t)b * p.c.kv_heads + h) * p.row_tiles + rt) * p.splits + split;
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;

  // ---- tile loads: thread owns chunk tid % (D/16) of keys tid / (D/16) + i * STEP
  constexpr int CPR = D / 16, STEP = KA_THREADS / CPR;
  const int ch = tid % CPR, key0 = tid / CPR;
  const int ppt = max(1, KT >> p.shift);  // pages per tile (KT >= 64; page 128: 1 and half used)
  int pid[4], spid = -1;
  auto load_ids = [&](int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = t * KT + key0 + i * STEP;
      pid[i] = key < kend ? kv8_page(table, p.c.max_pages, p.c.pages, key >> p.shift, nullptr) : -1;
    }
    if (tid < ppt) {
      const int key = t * KT + (tid << p.shift);
      spid = key < kend ? kv8_page(table, p.c.max_pages, p.c.pages, key >> p.shift, p.status) : -1;
    }
  };
  auto issue = [&](int t) {
    const int st = t % T::STAGES;
    uint8_t *kb = smem + st * 2 * KA_TILE, *vb = kb + KA_TILE;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (pid[i] < 0) continue;
      const int kl = key0 + i * STEP, key = t * KT + kl;
      const size_t off = (((size_t)pid[i] * p.c.kv_heads + h) * p.c.page +
                          (key & (p.c.page - 1))) * D + ch * 16;
      const uint32_t so = ka_chunk<D>(kl, ch);
      cp_async16(kb + so, p.c.k_codes + off);
      cp_async16(vb + so, p.c.v_codes + off);
    }
    if (tid < ppt) {
      // a page that is not there: K scale -1 masks its keys
      if (spid >= 0) {
        const size_t so = (size_t)spid * p.c.kv_heads + h;
        cp_async4(&s_ks[st][tid], p.c.k_scales + so);
        cp_async4(&s_vs[st][tid], p.c.v_scales + so);
      } else {
        s_ks[st][tid] = -1.f;
        s_vs[st][tid] = 0.f;
      }
    }
  };
#pragma unroll
  for (int s = 0; s < T::STAGES - 1; ++s) {
    if (t0 + s < t1) {
      load_ids(t0 + s);
      issue(t0 + s);
    }
    cp_async_commit();
  }
  if (t0 + T::STAGES - 1 < t1) load_ids(t0 + T::STAGES - 1);

  // ---- queries, in the order of the A fragments
  for (int r = warp; r < ROWS; r += 8) {
    const int R = r_base + r, i = R / p.rep, hr = R % p.rep;
    constexpr int PL = D / 32;  // elements per lane
    float x[PL];
    float amax = 0.f;
    const bool valid = t0 < t1 && R < rows && i < sp.q_len;
    const uint16_t *src = p.q + b * p.qb + (int64_t)(h * p.rep + hr) * p.qh + (int64_t)i * p.ql +
                          lane * PL;
    uint32_t w[PL / 2];
#pragma unroll
    for (int j = 0; j < PL / 2; ++j) w[j] = 0;
    if (valid) {
      if (p.vec) {
        if constexpr (PL == 8) {
          const uint4 v = ldg_v4(src);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (PL == 4) {
          const uint2 v = *reinterpret_cast<const uint2 *>(src);
          w[0] = v.x; w[1] = v.y;
        } else {
          w[0] = *reinterpret_cast<const uint32_t *>(src);
        }
      } else {
#pragma unroll
        for (int j = 0; j < PL / 2; ++j) w[j] = src[2 * j] | ((uint32_t)src[2 * j + 1] << 16);
      }
    }
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      x[j] = __uint_as_float((j & 1) ? (w[j >> 1] & 0xFFFF0000u) : (w[j >> 1] << 16));
      amax = fmaxf(amax, fabsf(x[j]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float pw = kv8_q_power(amax);
    if (lane == 0) s_fac[r] = p.scale_log2 / pw;
#pragma unroll
    for (int j = 0; j < PL; j += 2) {
      const int d = lane * PL + j, span = d >> 6, y = d & 15;
      const int fl = (r & 7) * 4 + ((d & 63) >> 4), reg = ((y & 2) ? 2 : 0) + ((r >> 3) & 1);
      uint32_t *dst = reinterpret_cast<uint32_t *>(
          s_q + ((r >> 4) * (D / 16) + span * 4 + (y >> 2)) * 32 + fl);
      dst[reg] = pack_h2(x[j] * pw, x[j + 1] * pw);
    }
  }

  int vis[MT][2];
  float fac[MT][2], m[MT][2], l[MT][2];
  float o[MT][4][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int R = r_base + mt * 16 + g + 8 * u;
      vis[mt][u] = R < rows ? sp.visible(R / p.rep) : 0;
      m[mt][u] = -INFINITY;
      l[mt][u] = 0.f;
    }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int u = 0; u < 4; ++u) o[mt][n][u] = 0.f;
  float vref = 0.f;
  const int kg = warp % T::NKG, dg = warp / T::NKG;
  __syncthreads();
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) fac[mt][u] = s_fac[mt * 16 + g + 8 * u];

  for (int t = t0; t < t1; ++t) {
    cp_async_wait<T::STAGES - 2>();
    __syncthreads();  // tile t is in; every warp is done with tile t - 1
    if (t + T::STAGES - 1 < t1) {
      issue(t + T::STAGES - 1);
      if (t + T::STAGES < t1) load_ids(t + T::STAGES);
    }
    cp_async_commit();
    const int st = t % T::STAGES;
    const uint8_t *kb = smem + st * 2 * KA_TILE, *vb = kb + KA_TILE;

    // ---- S = q K^T
    float acc[MT][T::NTW][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < T::NTW; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[mt][j][u] = 0.f;
#pragma unroll
    for (int s = 0; s < D / 64; ++s) {
      uint4 kw[T::NTW];
#pragma unroll
      for (int j = 0; j < T::NTW; ++j) {
        kw[j] = *reinterpret_cast<const uint4 *>(
            kb + ka_chunk<D>(8 * (warp * T::NTW + j) + g, 4 * s + c));
        kw[j].x ^= 0x80808080u; kw[j].y ^= 0x80808080u;
        kw[j].z ^= 0x80808080u; kw[j].w ^= 0x80808080u;
      }
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        uint4 a[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) a[mt] = s_q[(mt * (D / 16) + s * 4 + r4) * 32 + lane];
#pragma unroll
        for (int j = 0; j < T::NTW; ++j) {
          const uint32_t w = r4 == 0 ? kw[j].x : r4 == 1 ? kw[j].y : r4 == 2 ? kw[j].z : kw[j].w;
          const uint32_t b0 = h2_codes(__byte_perm(w, 0x64646464u, 0x4140));
          const uint32_t b1 = h2_codes(__byte_perm(w, 0x64646464u, 0x4342));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma_f16(acc[mt][j], a[mt], b0, b1);
        }
      }
    }

    // ---- scores, their maximum over the tile
    float vmax = 0.f;
    for (int i = 0; i < ppt; ++i) vmax = fmaxf(vmax, s_vs[st][i]);
    float tmax[MT][2], vfac[T::NTW];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) tmax[mt][0] = tmax[mt][1] = -INFINITY;
#pragma unroll
    for (int j = 0; j < T::NTW; ++j) {
      const int kl = 8 * (warp * T::NTW + j), pg = kl >> p.shift;
      const float ks = s_ks[st][pg];
      vfac[j] = s_vs[st][pg];
      const int key = t * KT + kl + 2 * c;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float z = acc[mt][j][u] * (fac[mt][u >> 1] * ks);
          acc[mt][j][u] = key + (u & 1) < vis[mt][u >> 1] && ks >= 0.f ? z : -INFINITY;
          tmax[mt][u >> 1] = fmaxf(tmax[mt][u >> 1], acc[mt][j][u]);
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x = tmax[mt][u];
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        if (c == 0) s_max[mt * 16 + g + 8 * u][warp] = x;
      }
    __syncthreads();

    // ---- weights as A fragments of the second product
    const float vnew = fmaxf(vref, vmax);
    const float vinv = vnew > 0.f ? 1.f / vnew : 0.f;
    const float vold = vref * vinv;
    vref = vnew;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float4 *mx = reinterpret_cast<const float4 *>(s_max[mt * 16 + g + 8 * u]);
        const float4 x = mx[0], y = mx[1];
        const float mn = fmaxf(fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)),
                                     fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w))), m[mt][u]);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = kv8_ex2(m[mt][u] - ref);
        m[mt][u] = mn;
        l[mt][u] *= alpha;
        const float ao = alpha * vold;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          o[mt][n][2 * u] *= ao;
          o[mt][n][2 * u + 1] *= ao;
        }
        const float sub = KV8_P_SHIFT - ref;
#pragma unroll
        for (int j = 0; j < T::NTW; ++j) {
          const float e0 = kv8_ex2(acc[mt][j][2 * u] + sub);
          const float e1 = kv8_ex2(acc[mt][j][2 * u + 1] + sub);
          l[mt][u] += e0 + e1;
          const float f = vfac[j] * vinv;
          const int nt = warp * T::NTW + j;  // 8-key group of the tile
          s_p[((mt * (KT / 16) + (nt >> 1)) * 32 + lane) * 4 + (nt & 1) * 2 + u] =
              pack_h2(e0 * f, e1 * f);
        }
      }
    __syncthreads();

    // ---- O += P V
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int ks = kg * 4 + s;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = ks * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
        w[i] = *reinterpret_cast<const uint32_t *>(
                   vb + ka_chunk<D>(key, 2 * dg + (g >> 2)) + (g & 3) * 4) ^ 0x80808080u;
      }
      uint4 a[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        a[mt] = *reinterpret_cast<const uint4 *>(s_p + ((mt * (KT / 16) + ks) * 32 + lane) * 4);
      const uint32_t x0 = __byte_perm(w[0], w[1], 0x5140), x1 = __byte_perm(w[0], w[1], 0x7362);
      const uint32_t y0 = __byte_perm(w[2], w[3], 0x5140), y1 = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t sel = (n & 1) ? 0x4342 : 0x4140;
        const uint32_t b0 = h2_codes(__byte_perm(n < 2 ? x0 : x1, 0x64646464u, sel));
        const uint32_t b1 = h2_codes(__byte_perm(n < 2 ? y0 : y1, 0x64646464u, sel));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mma_f16(o[mt][n], a[mt], b0, b1);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- sums over the warps: l over all eight, O over the key groups
  float *s_o = reinterpret_cast<float *>(smem);  // [NKG - 1][8 / NKG][ROWS][32]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x = l[mt][u];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (c == 0) s_l[warp][mt * 16 + g + 8 * u] = x;
    }
  constexpr int NDG = 8 / T::NKG;
  if (kg > 0) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float4 *d = reinterpret_cast<float4 *>(
            s_o + (((kg - 1) * NDG + dg) * ROWS + mt * 16 + g + 8 * u) * 32 + 8 * c);
        d[0] = make_float4(o[mt][0][2 * u], o[mt][1][2 * u], o[mt][2][2 * u], o[mt][3][2 * u]);
        d[1] = make_float4(o[mt][0][2 * u + 1], o[mt][1][2 * u + 1], o[mt][2][2 * u + 1],
                           o[mt][3][2 * u + 1]);
      }
  }
  __syncthreads();
  if (kg > 0) return;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = mt * 16 + g + 8 * u, R = r_base + r;
      if (R >= rows) continue;
      float f[8];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        f[n] = o[mt][n][2 * u];
        f[n + 4] = o[mt][n][2 * u + 1];
      }
#pragma unroll
      for (int k2 = 0; k2 < T::NKG - 1; ++k2) {
        const float4 *d = reinterpret_cast<const float4 *>(
            s_o + ((k2 * NDG + dg) * ROWS + r) * 32 + 8 * c);
        const float4 x = d[0], y = d[1];
        f[0] += x.x; f[1] += x.y; f[2] += x.z; f[3] += x.w;
        f[4] += y.x; f[5] += y.y; f[6] += y.z; f[7] += y.w;
      }
      float ls = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) ls += s_l[w][r];
      const int dim0 = 32 * dg + 8 * c;
      if (p.splits > 1) {
        if (dg == 0 && c == 0)
          p.ml_part[tile_id * ROWS + r] = make_float2(m[mt][u] - KV8_P_SHIFT, ls);
        if (t0 < t1) {
          float4 *dst = reinterpret_cast<float4 *>(p.o_part + (tile_id * ROWS + r) * D + dim0);
          dst[0] = make_float4(f[0] * vref, f[1] * vref, f[2] * vref, f[3] * vref);
          dst[1] = make_float4(f[4] * vref, f[5] * vref, f[6] * vref, f[7] * vref);
        }
      } else {
        const size_t row = ((size_t)b * p.Hq + h * p.rep + R % p.rep) * p.L + R / p.rep;
        const float inv = ls == 0.f ? 0.f : vref / ls;  // 0: the row sees no key
        *reinterpret_cast<uint4 *>(p.out + row * D + dim0) =
            make_uint4(pack_bf2(f[0] * inv, f[1] * inv), pack_bf2(f[2] * inv, f[3] * inv),
                       pack_bf2(f[4] * inv, f[5] * inv), pack_bf2(f[6] * inv, f[7] * inv));
        if (p.lse && dg == 0 && c == 0)
          p.lse[row] = ls == 0.f
                           ? -INFINITY
                           : (m[mt][u] - KV8_P_SHIFT + log2f(ls)) * 0.69314718055994531f;
      }
    }
}

// ------------------------------------------------------------------- combine
constexpr int KC_THREADS = 256;
constexpr int KC_MAX_SPLITS = 256;

// One CTA per output row: weights 2^(m_s - M) of the row's splits, then D / 4
// threads per split group add the splits in order and the groups are added in
// order.
template <int D>
__global__ void __launch_bounds__(KC_THREADS) kv8_combine_kernel(Kv8AttnParams p, int tile_rows) {
  __shared__ float s_w[KC_MAX_SPLITS];
  __shared__ float4 s_acc[KC_THREADS];
  __shared__ float s_red[KC_THREADS / 32], s_sum[KC_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rows = p.L * p.rep;
  const int R = blockIdx.x % rows, bh = blockIdx.x / rows;
  const size_t tile = ((size_t)bh * p.row_tiles + R / tile_rows) * p.splits;
  const int r = R % tile_rows;
  const float2 ml = tid < p.splits ? __ldcg(p.ml_part + (tile + tid) * tile_rows + r)
                                   : make_float2(-INFINITY, 0.f);
  float M = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KC_THREADS / 32; ++w) M = fmaxf(M, s_red[w]);
  const float wgt = ml.x == -INFINITY ? 0.f : kv8_ex2(ml.x - M);
  s_w[tid] = wgt;
  float ls = wgt * ml.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
  if ((tid & 31) == 0) s_sum[tid >> 5] = ls;
  __syncthreads();
  ls = 0.f;
#pragma unroll
  for (int w = 0; w < KC_THREADS / 32; ++w) ls += s_sum[w];
  constexpr int TPG = D / 4, G = KC_THREADS / TPG;
  const int d4 = tid % TPG, grp = tid / TPG;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = grp; s < p.splits; s += G) {
    const float w = s_w[s];
    if (w > 0.f) {  // a split without keys left no O
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(
                                  p.o_part + ((tile + s) * tile_rows + r) * D) + d4);
      a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y);
      a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w);
    }
  }
  s_acc[tid] = a;
  __syncthreads();
  if (grp > 0) return;
  for (int k = 1; k < G; ++k) {
    const float4 x = s_acc[k * TPG + d4];
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
  }
  const float inv = ls == 0.f ? 0.f : 1.f / ls;
  const int b = bh / p.c.kv_heads, h = bh % p.c.kv_heads;
  const size_t row = ((size_t)b * p.Hq + h * p.rep + R % p.rep) * p.L + R / p.rep;
  *(reinterpret_cast<uint2 *>(p.out + row * D) + d4) =
      make_uint2(pack_bf2(a.x * inv, a.y * inv), pack_bf2(a.z * inv, a.w * inv));
  if (p.lse && tid == 0)
    p.lse[row] =
        ls == 0.f ? -INFINITY : (M + log2f(ls)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------------- plan
struct Kv8Plan {
  int tile_rows, row_tiles, splits;
  bool tensor;
  size_t bytes;
};

// Up to 32 rows per kv head: kv8_attn_kernel, row tiles of 16 or 32 and two
// CTAs per SM; more rows: the tcgen05 kernel, one CTA per SM. Key ranges: as
// many as fill 148 SMs, and no more than there are tiles of keys in the table.
Kv8Plan kv8_plan(const VbKv8AttnArgs *a) {
  Kv8Plan pl;
  const long long rows = (long long)a->L * (a->q_heads / a->cache.kv_heads);
  pl.tensor = rows > 32;
  pl.tile_rows = pl.tensor ? kv8_prefill_rows(a->cache.dim) : rows <= 16 ? 16 : 32;
  pl.row_tiles = (int)((rows + pl.tile_rows - 1) / pl.tile_rows);
  const long long base = (long long)a->cache.batch * a->cache.kv_heads * pl.row_tiles;
  const long long kt = pl.tensor ? 128 : KA_TILE / a->cache.dim;
  const long long most = ((long long)a->cache.max_pages * a->cache.page + kt - 1) / kt;
  long long s = (pl.tensor ? 148 : 2 * 148) / base;
  s = s < 1 ? 1 : s > most ? most : s;
  pl.splits = (int)(s > KC_MAX_SPLITS ? KC_MAX_SPLITS : s);
  pl.bytes = pl.splits == 1 ? 0
                            : (size_t)base * pl.splits * pl.tile_rows * (a->cache.dim + 2) * 4;
  return pl;
}

template <int D, int MT>
int kv8_launch(const Kv8AttnParams &p, cudaStream_t s) {
  using T = Kv8Tile<D, MT>;
  static bool ready = false;
  if (!ready) {
    const cudaError_t e = cudaFuncSetAttribute(
        kv8_attn_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != cudaSuccess)
      return set_error(VB_ERR_CUDA, "kv8_attn_kernel attributes: %s", cudaGetErrorString(e));
    ready = true;
  }
  vb_launch(kv8_attn_kernel<D, MT>, dim3(p.splits, p.c.kv_heads * p.row_tiles, p.c.batch),
            dim3(KA_THREADS), T::SMEM, s, false, p);
  return check_launch("kv8_attn_kernel");
}

template <int D>
int kv8_run(const Kv8AttnParams &p, const Kv8Plan &pl, cudaStream_t s) {
  const int rc = pl.tensor ? kv8_prefill_launch(p, s)
                 : pl.tile_rows == 16 ? kv8_launch<D, 1>(p, s)
                                      : kv8_launch<D, 2>(p, s);
  if (rc != VB_OK || p.splits == 1) return rc;
  vb_launch(kv8_combine_kernel<D>, dim3(p.c.batch * p.c.kv_heads * p.L * p.rep),
            dim3(KC_THREADS), 0, s, true, p, pl.tile_rows);
  return check_launch("kv8_combine_kernel");
}

int kv8_attn_check(const VbKv8AttnArgs *a) {
  VB_REQUIRE(a, "vb_kv8_attn: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_attn");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->q_heads >= 1 && a->q_heads % a->cache.kv_heads == 0 &&
                 a->q_heads / a->cache.kv_heads <= 128,
             "vb_kv8_attn: %d query heads over %d kv heads (at most 128 each)", a->q_heads,
             a->cache.kv_heads);
  VB_REQUIRE(a->L >= 0 && (long long)a->L * a->q_heads <= 1 << 26,
             "vb_kv8_attn: L=%d rows of %d heads", a->L, a->q_heads);
  return VB_OK;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

size_t vb_kv8_attn_workspace_size(const VbKv8AttnArgs *a) {
  if (kv8_attn_check(a) != VB_OK || a->L == 0) return 0;
  return kv8_plan(a).bytes;
}

int vb_kv8_attn(const VbKv8AttnArgs *a, vb_stream_t stream) {
  const int rc = kv8_attn_check(a);
  if (rc != VB_OK) return rc;
  if (a->L == 0) return VB_OK;
  VB_REQUIRE(a->q && a->lens && a->out, "vb_kv8_attn: null tensor");
  VB_REQUIRE(((uintptr_t)a->out % 16) == 0, "vb_kv8_attn: out must be 16-byte aligned");
  VB_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "vb_kv8_attn: scale %g", (double)a->scale);
  const Kv8Plan pl = kv8_plan(a);
  if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes))
    return set_error(VB_ERR_WORKSPACE, "vb_kv8_attn: workspace %zu < %zu bytes",
                     a->workspace_bytes, pl.bytes);
  VB_REQUIRE(((uintptr_t)a->workspace % 16) == 0, "vb_kv8_attn: workspace alignment");
  VB_REQUIRE((long long)a->cache.kv_heads * pl.row_tiles <= 65535 &&
                 (long long)a->cache.batch * a->q_heads * a->L <= 0x7fffffffll,
             "vb_kv8_attn: too many rows");
  Kv8AttnParams p;
  p.c = a->cache;
  p.q = a->q;
  p.qb = a->q_strides[0]; p.qh = a->q_strides[1]; p.ql = a->q_strides[2];
  p.lens = a->lens; p.q_lens = a->q_lens;
  p.out = a->out; p.lse = a->lse; p.status = a->status;
  p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
  p.Hq = a->q_heads; p.L = a->L; p.rep = a->q_heads / a->cache.kv_heads;
  p.len_add = a->len_add; p.causal = a->causal ? 1 : 0;
  p.shift = kv8_page_shift(a->cache.page);
  p.vec = ((uintptr_t)a->q % 16) == 0 && p.qb % 8 == 0 && p.qh % 8 == 0 && p.ql % 8 == 0;
  p.row_tiles = pl.row_tiles; p.splits = pl.splits;
  p.o_part = static_cast<float *>(a->workspace);
  p.ml_part = reinterpret_cast<float2 *>(
      p.o_part + (size_t)a->cache.batch * a->cache.kv_heads * pl.row_tiles * pl.splits *
                     pl.tile_rows * a->cache.dim);
  cudaStream_t s = as_stream(stream);
  switch (a->cache.dim) {
    case 64: return kv8_run<64>(p, pl, s);
    case 128: return kv8_run<128>(p, pl, s);
    default: return kv8_run<256>(p, pl, s);
  }
}

}  // extern "C"
