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
// A CTA (8 warps) owns an equal share of all sequences' key tiles (16 KB of K
// and of V each) and all query rows, up to 32, of the kv head it is at. cp.async
// brings the tiles into a ring (the rows
// of a page are contiguous; chunks of 16 bytes are XOR-swizzled so that both
// fragment reads below are free of bank conflicts):
//   S: warp w takes 2048 / D keys of the tile over all of D; lane (g, c) of an
//      8-key group reads 16 consecutive bytes of key g, four k-steps of the
//      product (the order of dims within a 64-dim span is the same permutation
//      for q);
//   max over the warps through shared memory, weights as PV's A fragments;
//   PV: warp takes 32 dims and four 16-key steps; lane (g, c) reads 4 bytes of
//      its four keys and interleaves them into key pairs.
// Shares of one (sequence, kv head) meet in kv8_combine_kernel.
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

// ------------------------------------------------------------ work partition
// The key tiles of all (sequence, kv head) units in one row, [0, total), are
// dealt to the CTAs in equal contiguous ranges, whatever the sequences'
// lengths. A unit that lies in one CTA's range is finished there; the others
// leave at most two partial results per CTA: slot 1 for a unit that begins in
// the range, slot 0 for one that began before it.
struct Kv8Deal {
  unsigned long long total, q;
  uint32_t r;
  __device__ Kv8Deal(unsigned long long t, uint32_t ctas) : total(t) {
    if ((t >> 32) == 0) {
      q = (uint32_t)t / ctas;
      r = (uint32_t)t % ctas;
    } else {
      q = t / ctas;
      r = (uint32_t)(t % ctas);
    }
  }
  __device__ unsigned long long begin(uint32_t c) const { return c * q + min(c, r); }
  __device__ uint32_t owner(unsigned long long x) const {  // x < total
    const unsigned long long big = (q + 1) * r;
    return x < big ? (uint32_t)(x / (q + 1)) : r + (uint32_t)((x - big) / q);
  }
};

// Key tiles of sequence b.
template <int KT>
__device__ __forceinline__ int kv8_tiles(const Kv8AttnParams &p, int b, bool flag) {
  const Kv8Span sp = kv8_span(p, b, flag);
  return sp.q_len > 0 ? (sp.visible(sp.q_len - 1) + KT - 1) / KT : 0;
}

// Tiles of all sequences together; every thread of the CTA gets it.
template <int KT>
__device__ __forceinline__ unsigned long long kv8_all_tiles(const Kv8AttnParams &p, bool flag,
                                                            unsigned long long *s_sum) {
  if (p.c.batch == 1) return kv8_tiles<KT>(p, 0, flag && threadIdx.x == 0);
  unsigned long long y = 0;
  for (int b = threadIdx.x; b < p.c.batch; b += KA_THREADS) y += kv8_tiles<KT>(p, b, flag);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = y;
  __syncthreads();
  y = 0;
#pragma unroll
  for (int w = 0; w < KA_THREADS / 32; ++w) y += s_sum[w];
  return y;
}

template <int D, int MT>
__global__ void __launch_bounds__(KA_THREADS, 2) kv8_attn_kernel(Kv8AttnParams p) {
  using T = Kv8Tile<D, MT>;
  constexpr int KT = T::KT, ROWS = 16 * MT;
  extern __shared__ __align__(128) uint8_t smem[];
  uint4 *s_q = reinterpret_cast<uint4 *>(smem + T::RING);                // [MT][D/16][32]
  uint32_t *s_p = reinterpret_cast<uint32_t *>(smem + T::RING + T::Q_BYTES);  // [MT][KT/16][32][4]
  __shared__ __align__(16) float s_max[ROWS][8];
  __shared__ float s_fac[ROWS], s_l[8][ROWS];
  __shared__ unsigned long long s_sum[KA_THREADS / 32], s_begin;
  __shared__ int s_b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const int H = p.c.kv_heads, rows = p.L * p.rep;

  // ---- this CTA's tiles, and the sequence its range begins in
  const Kv8Deal deal(kv8_all_tiles<KT>(p, blockIdx.x == 0, s_sum) * H, gridDim.x);
  unsigned long long w0 = deal.begin(blockIdx.x);
  const unsigned long long w1 = deal.begin(blockIdx.x + 1);
  if (w0 == w1) return;
  int b = 0;
  unsigned long long b_begin = 0;  // tiles of the sequences before b, all heads
  if (p.c.batch > 1) {
    if (warp == 0) {  // 32 sequences at a time
      for (int b0 = 0; b0 < p.c.batch; b0 += 32) {
        unsigned long long n = b0 + lane < p.c.batch
                                   ? (unsigned long long)kv8_tiles<KT>(p, b0 + lane, false) * H : 0;
        unsigned long long inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, b_begin + inc > w0);
        if (hit) {
          const int at = __ffs(hit) - 1;
          const unsigned long long start = b_begin + __shfl_sync(0xffffffffu, inc - n, at);
          if (lane == 0) {
            s_b = b0 + at;
            s_begin = start;
          }
          break;
        }
        b_begin += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    __syncthreads();
    b = s_b;
    b_begin = s_begin;
  }

  // thread owns chunk tid % (D/16) of keys tid / (D/16) + i * STEP of a tile
  constexpr int CPR = D / 16, STEP = KA_THREADS / CPR, NG = KT / 16;
  const int ch = tid % CPR, key0 = tid / CPR;
  const uint32_t pool_step = (uint32_t)(H * p.c.page * D);
  const int kg = warp % T::NKG, dg = warp / T::NKG;

  while (w0 < w1) {
    // ---- the unit at w0: sequence b, head h, tiles [t0, t1) of `tiles`
    const Kv8Span sp = kv8_span(p, b, false);
    const int kend = sp.q_len > 0 ? sp.visible(sp.q_len - 1) : 0;
    const int tiles = (kend + KT - 1) / KT;
    const unsigned long long off = w0 - b_begin;
    if (off >= (unsigned long long)tiles * H) {  // past this sequence
      b_begin += (unsigned long long)tiles * H;
      ++b;
      continue;
    }
    const int h = (int)(off >> 32 ? off / tiles : (uint32_t)off / (uint32_t)tiles);
    const int t0 = (int)(off - (unsigned long long)h * tiles);
    const int t1 = (int)min((unsigned long long)tiles, t0 + (w1 - w0));
    if (t0 == 0 && tid == 0)  // the CTAs that share this unit, for the combine kernel
      p.units[b * H + h] =
          make_int2(blockIdx.x, (int)(deal.owner(w0 + tiles - 1) - blockIdx.x) + 1);
    w0 += t1 - t0;
    const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
    const int8_t *kbase = p.c.k_codes + (size_t)h * p.c.page * D + ch * 16;
    const int8_t *vbase = p.c.v_codes + (size_t)h * p.c.page * D + ch * 16;

    // Page of the 16-key group lane % NG of a tile; -1: none (past the last key,
    // or flagged). Such rows read page 0 and get no weight.
    auto group_page = [&](int t) {
      const int key = t * KT + (lane % NG) * 16;
      return t < t1 && key < kend
                 ? kv8_page(table, p.c.max_pages, p.c.pages, key >> p.shift, p.status) : -1;
    };
    // K scale of the group (-1 masks it) and V scale
    auto group_scales = [&](int id, float &ks, float &vs) {
      ks = id >= 0 ? __ldg(p.c.k_scales + (size_t)id * H + h) : -1.f;
      vs = id >= 0 ? __ldg(p.c.v_scales + (size_t)id * H + h) : 0.f;
    };
    auto issue = [&](int t, int id) {
      uint8_t *kb = smem + (t % T::STAGES) * 2 * KA_TILE, *vb = kb + KA_TILE;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kl = key0 + i * STEP;
        const uint32_t pg = (uint32_t)max(0, __shfl_sync(0xffffffffu, id, kl >> 4));
        const unsigned long long at = (unsigned long long)pg * pool_step +
                                      ((t * KT + kl) & (p.c.page - 1)) * D;
        const uint32_t so = ka_chunk<D>(kl, ch);
        cp_async16(kb + so, kbase + at);
        cp_async16(vb + so, vbase + at);
      }
    };
    int id_next = group_page(t0);
    float ks_l, vs_l;
    group_scales(id_next, ks_l, vs_l);
#pragma unroll
    for (int s = 0; s < T::STAGES - 1; ++s) {
      if (t0 + s < t1) issue(t0 + s, id_next);
      cp_async_commit();
      id_next = group_page(t0 + s + 1);
    }
    // scales run one tile ahead of their use, page numbers with the copies
    int id_scale = T::STAGES == 2 ? id_next : group_page(t0 + 1);

    // ---- queries, in the order of the A fragments
    for (int r = warp; r < ROWS; r += 8) {
      const int i = p.row_of(r), hr = r - i * p.rep;
      constexpr int PL = D / 32;  // elements per lane
      float x[PL];
      float amax = 0.f;
      const uint16_t *src = p.q + b * p.qb + (int64_t)(h * p.rep + hr) * p.qh +
                            (int64_t)i * p.ql + lane * PL;
      uint32_t w[PL / 2];
#pragma unroll
      for (int j = 0; j < PL / 2; ++j) w[j] = 0;
      if (r < rows && i < sp.q_len) {
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
      amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
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
        const int r = mt * 16 + g + 8 * u;
        vis[mt][u] = r < rows ? sp.visible(p.row_of(r)) : 0;
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
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) fac[mt][u] = s_fac[mt * 16 + g + 8 * u];

    for (int t = t0; t < t1; ++t) {
      cp_async_wait<T::STAGES - 2>();
      __syncthreads();  // tile t is in; every warp is done with tile t - 1
      if (t + T::STAGES - 1 < t1) {
        issue(t + T::STAGES - 1, id_next);
        id_next = group_page(t + T::STAGES);
      }
      cp_async_commit();
      float ks_n, vs_n;  // of tile t + 1
      group_scales(id_scale, ks_n, vs_n);
      id_scale = group_page(t + 2);
      const uint8_t *kb = smem + (t % T::STAGES) * 2 * KA_TILE, *vb = kb + KA_TILE;

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
      float vmax = vs_l;
#pragma unroll
      for (int o2 = NG / 2; o2 > 0; o2 >>= 1)
        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o2));
      float tmax[MT][2], vfac[T::NTW];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) tmax[mt][0] = tmax[mt][1] = -INFINITY;
#pragma unroll
      for (int j = 0; j < T::NTW; ++j) {
        const int kl = 8 * (warp * T::NTW + j);
        const float ks = __shfl_sync(0xffffffffu, ks_l, kl >> 4);
        vfac[j] = __shfl_sync(0xffffffffu, vs_l, kl >> 4);
        const int key = ks < 0.f ? 0x7fffffff - 64 : t * KT + kl + 2 * c;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float z = acc[mt][j][u] * (fac[mt][u >> 1] * ks);
            acc[mt][j][u] = key + (u & 1) < vis[mt][u >> 1] ? z : -INFINITY;
            tmax[mt][u >> 1] = fmaxf(tmax[mt][u >> 1], acc[mt][j][u]);
          }
      }
      ks_l = ks_n;
      vs_l = vs_n;
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
      const float vinv = vnew > 0.f ? __frcp_rn(vnew) : 0.f;
      const float vold = vref * vinv;
      vref = vnew;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float sub[2];
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
          sub[u] = KV8_P_SHIFT - ref;
        }
#pragma unroll
        for (int j = 0; j < T::NTW; ++j) {
          const float f = vfac[j] * vinv;
          uint32_t pk[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float e0 = kv8_ex2(acc[mt][j][2 * u] + sub[u]);
            const float e1 = kv8_ex2(acc[mt][j][2 * u + 1] + sub[u]);
            l[mt][u] += e0 + e1;
            pk[u] = pack_h2(e0 * f, e1 * f);
          }
          const int nt = warp * T::NTW + j;  // 8-key group of the tile
          *reinterpret_cast<uint2 *>(
              s_p + ((mt * (KT / 16) + (nt >> 1)) * 32 + lane) * 4 + (nt & 1) * 2) =
              make_uint2(pk[0], pk[1]);
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
    if (kg == 0) {
      const bool whole = t0 == 0 && t1 == tiles;
      const size_t slot = (size_t)blockIdx.x * 2 + (t0 == 0);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = mt * 16 + g + 8 * u;
          if (r >= rows) continue;
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
          if (!whole) {
            if (dg == 0 && c == 0)
              p.ml_part[slot * ROWS + r] = make_float2(m[mt][u] - KV8_P_SHIFT, ls);
            float4 *dst = reinterpret_cast<float4 *>(p.o_part + (slot * ROWS + r) * D + dim0);
            dst[0] = make_float4(f[0] * vref, f[1] * vref, f[2] * vref, f[3] * vref);
            dst[1] = make_float4(f[4] * vref, f[5] * vref, f[6] * vref, f[7] * vref);
          } else {
            const int i = p.row_of(r);
            const size_t row = ((size_t)b * p.Hq + h * p.rep + r - i * p.rep) * p.L + i;
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
    if (w0 < w1) __syncthreads();  // the ring, s_q and s_l are free for the next unit
  }
}

// ------------------------------------------------------------------- combine
constexpr int KC_MAX = 512;  // most partial results of one row

// Where a row's partial results are. kv8_attn_kernel's units (`units` not
// null): slot 1 of the first CTA that shares the unit, slot 0 of the following
// ones; n = 1: finished by that CTA, n = 0: a sequence without keys, whose
// zeros are written here. The prefill kernel: `splits` per row tile.
struct Kv8Parts {
  int n;
  size_t first, step, skip;
  __device__ size_t at(int s) const { return first + s * step - (s > 0 ? skip : 0); }
};
template <int D>
__device__ __forceinline__ Kv8Parts kv8_parts(const Kv8AttnParams &p, int bh, int b, int tile) {
  Kv8Parts q;
  if (p.units) {
    const int2 u = __ldcg(p.units + bh);  // (left from an earlier call if there are no tiles)
    const int tiles = kv8_tiles<KA_TILE / D>(p, b, false);
    q.n = tiles > 0 ? u.y : 0;
    q.first = (size_t)u.x * 2 + 1;
    q.step = 2;
    q.skip = 1;
  } else {
    q.n = p.splits;
    q.first = ((size_t)bh * p.row_tiles + tile) * p.splits;
    q.step = 1;
    q.skip = 0;
  }
  return q;
}
__device__ __forceinline__ void kv8_finish(const Kv8AttnParams &p, int D, int b, int h, int R,
                                           int d4, float M, float ls, float4 a) {
  const int i = p.row_of(R);
  const size_t row = ((size_t)b * p.Hq + h * p.rep + R - i * p.rep) * p.L + i;
  const float inv = ls == 0.f ? 0.f : 1.f / ls;
  *(reinterpret_cast<uint2 *>(p.out + row * D) + d4) =
      make_uint2(pack_bf2(a.x * inv, a.y * inv), pack_bf2(a.z * inv, a.w * inv));
  if (p.lse && d4 == 0)
    p.lse[row] = ls == 0.f ? -INFINITY : (M + log2f(ls)) * 0.69314718055994531f;
}

// Joins the partial results of rows: weights 2^(m_s - M), O and l summed over
// them in order. For few partial results per row a thread joins four dims of
// one row.
template <int D>
__global__ void __launch_bounds__(KA_THREADS) kv8_combine_kernel(Kv8AttnParams p, int tile_rows) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int RPC = KA_THREADS * 4 / D;  // rows per CTA
  const int rows = p.L * p.rep, groups = (rows + RPC - 1) / RPC;
  const int bh = blockIdx.x / groups, R = blockIdx.x % groups * RPC + threadIdx.x / (D / 4);
  const int b = bh / p.c.kv_heads, h = bh % p.c.kv_heads, d4 = threadIdx.x % (D / 4);
  if (R >= rows) return;
  const Kv8Parts q = kv8_parts<D>(p, bh, b, R / tile_rows);
  if (p.units && q.n == 1) return;
  const int r = R % tile_rows;
  float M = -INFINITY, ls = 0.f;
#pragma unroll 4
  for (int s = 0; s < q.n; ++s) M = fmaxf(M, __ldcg(p.ml_part + q.at(s) * tile_rows + r).x);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < q.n; ++s) {
    const size_t at = q.at(s) * tile_rows + r;
    const float2 ml = __ldcg(p.ml_part + at);
    const float w = ml.x == -INFINITY ? 0.f : kv8_ex2(ml.x - M);
    ls = fmaf(w, ml.y, ls);
    if (w > 0.f) {  // a range without visible keys left no O
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(p.o_part + at * D) + d4);
      a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y);
      a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w);
    }
  }
  kv8_finish(p, D, b, h, R, d4, M, ls, a);
}

// For many partial results per row: a CTA takes 32 dims of one row, 8 threads
// per partial result and 32 of them at a time, so that all loads are in flight
// at once.
template <int D>
__global__ void __launch_bounds__(KA_THREADS) kv8_combine_wide_kernel(Kv8AttnParams p,
                                                                      int tile_rows) {
  __shared__ float s_w[KC_MAX];
  __shared__ float4 s_acc[KA_THREADS];
  __shared__ float s_red[KA_THREADS / 32], s_ls[KA_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rows = p.L * p.rep;
  const int R = blockIdx.x % rows, bh = blockIdx.x / rows;
  const int b = bh / p.c.kv_heads, h = bh % p.c.kv_heads;
  const int d4 = blockIdx.y * 8 + (tid & 7), grp = tid >> 3, r = R % tile_rows;
  const Kv8Parts q = kv8_parts<D>(p, bh, b, R / tile_rows);
  if (p.units && q.n == 1) return;
  float M = -INFINITY, ls = 0.f;
  float2 ml[KC_MAX / KA_THREADS];
#pragma unroll
  for (int k = 0; k < KC_MAX / KA_THREADS; ++k) {
    const int s = tid + k * KA_THREADS;
    ml[k] = s < q.n ? __ldcg(p.ml_part + q.at(s) * tile_rows + r) : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[k].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KA_THREADS / 32; ++w) M = fmaxf(M, s_red[w]);
#pragma unroll
  for (int k = 0; k < KC_MAX / KA_THREADS; ++k) {
    const float wgt = ml[k].x == -INFINITY ? 0.f : kv8_ex2(ml[k].x - M);
    s_w[tid + k * KA_THREADS] = wgt;
    ls = fmaf(wgt, ml[k].y, ls);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
  if ((tid & 31) == 0) s_ls[tid >> 5] = ls;
  __syncthreads();
  ls = 0.f;
#pragma unroll
  for (int w = 0; w < KA_THREADS / 32; ++w) ls += s_ls[w];
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = grp; s < q.n; s += 32) {
    const float w = s_w[s];
    if (w > 0.f) {
      const float4 x =
          __ldcg(reinterpret_cast<const float4 *>(p.o_part + (q.at(s) * tile_rows + r) * D) + d4);
      a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y);
      a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w);
    }
  }
  s_acc[tid] = a;
  __syncthreads();
  if (tid >= 8) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) {
    const float4 x = s_acc[k * 8 + tid];
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
  }
  kv8_finish(p, D, b, h, R, d4, M, ls, a);
}

// ---------------------------------------------------------------------- plan
struct Kv8Plan {
  int tile_rows, row_tiles, splits, ctas;
  bool tensor;
  size_t parts, bytes;  // partial results (tile_rows rows each), workspace
  bool wide;            // many partial results per row
};

// Up to 32 rows per kv head: kv8_attn_kernel, row tiles of 16 or 32, two CTAs
// on each of 148 SMs (fewer when the table holds fewer tiles). More rows: the
// tcgen05 kernel, one CTA per SM, key ranges as many as fill 148 SMs.
Kv8Plan kv8_plan(const VbKv8AttnArgs *a) {
  Kv8Plan pl;
  const long long rows = (long long)a->L * (a->q_heads / a->cache.kv_heads);
  const long long units = (long long)a->cache.batch * a->cache.kv_heads;
  const long long cap = (long long)a->cache.max_pages * a->cache.page;
  pl.tensor = rows > 32;
  if (pl.tensor) {
    pl.tile_rows = kv8_prefill_rows(a->cache.dim);
    pl.row_tiles = (int)((rows + pl.tile_rows - 1) / pl.tile_rows);
    const long long base = units * pl.row_tiles, most = (cap + 127) / 128;
    long long s = 148 / base;
    s = s < 1 ? 1 : s > most ? most : s;
    pl.splits = (int)s;
    pl.ctas = 0;
    pl.parts = s == 1 ? 0 : (size_t)(base * s);
  } else {
    pl.tile_rows = rows <= 16 ? 16 : 32;
    pl.row_tiles = pl.splits = 1;
    const long long kt = KA_TILE / a->cache.dim, tiles = units * ((cap + kt - 1) / kt);
    pl.ctas = (int)(tiles < 2 * 148 ? tiles : 2 * 148);
    pl.parts = (size_t)pl.ctas * 2;
  }
  // results per row on average: the wide kernel pays from about 8
  pl.wide = pl.tensor ? pl.splits > 8 : pl.ctas > 8 * units;
  pl.bytes = pl.parts * pl.tile_rows * (a->cache.dim + 2) * sizeof(float) +
             (pl.tensor ? 0 : units * sizeof(int2));
  return pl;
}

template <int D, int MT>
int kv8_launch(const Kv8AttnParams &p, int ctas, cudaStream_t s) {
  using T = Kv8Tile<D, MT>;
  static bool ready = false;
  if (!ready) {
    const cudaError_t e = cudaFuncSetAttribute(
        kv8_attn_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != cudaSuccess)
      return set_error(VB_ERR_CUDA, "kv8_attn_kernel attributes: %s", cudaGetErrorString(e));
    ready = true;
  }
  vb_launch(kv8_attn_kernel<D, MT>, dim3(ctas), dim3(KA_THREADS), T::SMEM, s, false, p);
  return check_launch("kv8_attn_kernel");
}

template <int D>
int kv8_run(const Kv8AttnParams &p, const Kv8Plan &pl, cudaStream_t s) {
  const int rc = pl.tensor ? kv8_prefill_launch(p, s)
                 : pl.tile_rows == 16 ? kv8_launch<D, 1>(p, pl.ctas, s)
                                      : kv8_launch<D, 2>(p, pl.ctas, s);
  if (rc != VB_OK || pl.parts == 0) return rc;
  const unsigned units = p.c.batch * p.c.kv_heads, rows = p.L * p.rep;
  constexpr unsigned RPC = KA_THREADS * 4 / D;
  if (pl.wide)
    vb_launch(kv8_combine_wide_kernel<D>, dim3(units * rows, D / 32), dim3(KA_THREADS), 0, s, true,
              p, pl.tile_rows);
  else
    vb_launch(kv8_combine_kernel<D>, dim3(units * ((rows + RPC - 1) / RPC)), dim3(KA_THREADS), 0, s,
              true, p, pl.tile_rows);
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
  VB_REQUIRE(a->L >= 0 && (long long)a->L * a->q_heads <= 1 << 24,
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
  p.rep_inv = (uint32_t)((1ull << 32) / (uint32_t)p.rep) + (p.rep > 1);
  p.o_part = static_cast<float *>(a->workspace);
  p.ml_part = reinterpret_cast<float2 *>(p.o_part + pl.parts * pl.tile_rows * a->cache.dim);
  p.units = pl.tensor ? nullptr
                      : reinterpret_cast<int2 *>(p.ml_part + pl.parts * pl.tile_rows);
  cudaStream_t s = as_stream(stream);
  switch (a->cache.dim) {
    case 64: return kv8_run<64>(p, pl, s);
    case 128: return kv8_run<128>(p, pl, s);
    default: return kv8_run<256>(p, pl, s);
  }
}

}  // extern "C"
