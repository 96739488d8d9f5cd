// Attention over the paged 8-bit KV cache, few query rows per kv head (decode
// and verify steps): HBM-bound, one byte per cached value.
//
//   z = scale * s_K(page) * (q . code_K),  o = sum_j 2^(z_j log2 e - m) s_V(page_j) code_V / l
//
// The codes are exact in f16 and so are the queries after a power of two per
// row, so q . code runs on f16 tensor-core products with float32 sums; the
// scales are applied to the sums. The weights are rounded to f16 (11 bits)
// after a factor s_V(page) / v, v the largest V scale so far: the codes are f16, so the
// weights have to be; an eighth of what out loses to bf16. l is summed in float32
// from the unrounded weights.
//
// A CTA (4 warps, two or three CTAs per SM) owns an equal share of all sequences' key
// tiles (16 KB of K and of V each) and all query rows, up to 32, of the kv head
// it is at. cp.async brings the tiles into a ring (the rows of a page are
// contiguous; chunks of 16 bytes are XOR-swizzled so that both fragment reads
// below are free of bank conflicts). Both products are transposed, so that rows
// come in eights and a converted K or V fragment serves every group of rows:
//   S^T = K q^T: a warp takes 4096 / D keys; lane (g, c) reads 16 consecutive
//      bytes of keys g and g + 8, four k-steps of the product (the order of
//      dims within a 64-dim span is the same permutation for q);
//   O^T += V^T P^T: a warp takes D / 4 dims of every key; lane (g, c) reads 4
//      bytes of its four keys and interleaves them into key pairs.
// The running maximum and the largest V scale only move when a score passes the
// maximum by 2^2 or a tile brings a larger scale: all warps then meet, take the
// new values and form the weights again. Otherwise the weights stand as
// they are and a tile costs two barriers.
// Shares of one (sequence, kv head) are joined by the last of its CTAs to finish
// (ticket), or, when there are few units, by kv8_combine_wide_kernel.
//
// What bounds it: one row over 131,072 keys, 16/2 heads of 256, takes 37.7 us for 134
// MB (3.6 TB/s; a copy 20.8): in the middle HBM is at 0.85 of a copy, the start and
// the joining of 222 partial results take the rest. 16 sequences x 4 rows over up to
// 8,190 keys, 32/8 heads of 128: 49 us for 127 MB (a copy 19.7), bound by latency:
// with the 12 warps that registers and the rings leave room for, issue slots are half
// used and HBM at a third; warps wait for products, shared memory and each other. With
// 32 rows (8 warps): 16 sequences of 8,190 keys 103 us for 268 MB.
#include "kv8_attn.cuh"

namespace vb {
namespace {

constexpr int KA_THREADS = 128;
constexpr int KA_TILE = 16384;          // bytes of K, and of V, per tile
constexpr int KA_STAGES = 2;
constexpr int KA_TICKETS = 16384;       // units that a ticket word can join
static_assert(KA_TICKETS * sizeof(uint32_t) == VB_KV8_ATTN_WORKSPACE_HEAD, "ticket words");
// Weights as f16 are 2^(z - m) s_V / v with m the row's maximum less KA_SHIFT, until
// the maximum has grown by more than KA_MOVE: at most 2^15. m is rounded up and what a
// score may reach down, so that this holds for scores of any size.
constexpr float KA_SHIFT = 13.f;
constexpr float KA_MOVE = 2.f;

template <int D, int NR>  // NR groups of 8 query rows
struct Kv8Tile {
  static constexpr int KT = KA_TILE / D;     // keys per tile
  static constexpr int CTAS = NR > 2 ? 2 : 3;  // per SM (shared memory, registers)
  static constexpr int MW = KT / 64;         // 16-key groups per warp (S)
  static constexpr int DW = D / 4;           // dims per warp (PV)
  static constexpr int ND = DW >= 32 ? DW / 32 : 1;  // 32-dim groups per warp (16 dims: D = 64)
  static constexpr int NM = DW / 16;         // 16-dim fragments per warp
  static constexpr int RING = KA_STAGES * 2 * KA_TILE;
  static constexpr int Q_BYTES = NR * D * 16;
  static constexpr int P_BYTES = NR * KT * 16;
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
    if ((total >> 32) == 0)
      return x < big ? (uint32_t)x / (uint32_t)(q + 1)
                     : r + (uint32_t)(x - big) / (uint32_t)q;
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

// Writes four dims of an output row: a / ls (0 for a row that saw no key).
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

// Joins four dims of a row: the partial results at(0) .. at(n - 1) (rows of O
// and of (m, l)), weights 2^(m_s - M), summed in order.
template <int D, typename At>
__device__ __forceinline__ void kv8_join(const Kv8AttnParams &p, int b, int h, int R, int d4,
                                         int n, At at) {
  float M = -INFINITY, ls = 0.f;
#pragma unroll 8
  for (int s = 0; s < n; ++s) M = fmaxf(M, __ldcg(p.ml_part + at(s)).x);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < n; ++s) {
    const float2 ml = __ldcg(p.ml_part + at(s));
    const float4 x = __ldcg(reinterpret_cast<const float4 *>(p.o_part + at(s) * D) + d4);
    const float w = ml.x == -INFINITY ? 0.f : kv8_ex2(ml.x - M);
    ls = fmaf(w, ml.y, ls);
    if (w > 0.f) {  // a range without visible keys left no O
      a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y);
      a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w);
    }
  }
  kv8_finish(p, D, b, h, R, d4, M, ls, a);
}

__device__ __forceinline__ void ldsm_x2_trans(uint32_t &r0, uint32_t &r1, const void *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r0), "=r"(r1)
               : "r"((uint32_t)__cvta_generic_to_shared(p)));
}

template <int D, int NR>
__global__ void __launch_bounds__(KA_THREADS, Kv8Tile<D, NR>::CTAS) kv8_attn_kernel(Kv8AttnParams p) {
  using T = Kv8Tile<D, NR>;
  constexpr int KT = T::KT, ROWS = 8 * NR, MW = T::MW, NM = T::NM;
  extern __shared__ __align__(128) uint8_t smem[];
  uint32_t *s_q = reinterpret_cast<uint32_t *>(smem + T::RING);  // [NR][D/32][32 lanes][4]
  uint8_t *s_p = smem + T::RING + T::Q_BYTES;                    // f16 [NR][KT keys][8 rows]
  __shared__ float s_fac[ROWS], s_max[4][ROWS], s_l[4][ROWS];
  __shared__ unsigned long long s_sum[KA_THREADS / 32], s_begin;
  __shared__ int s_b, s_move[2], s_share[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  const int H = p.c.kv_heads, rows = p.L * p.rep;

  // ---- rows of sequences without visible keys
  for (int z = blockIdx.x; z < p.c.batch; z += gridDim.x) {
    if (kv8_tiles<KT>(p, z, false) > 0) continue;
    const size_t row0 = (size_t)z * p.Hq * p.L, n = (size_t)p.Hq * p.L;
    for (size_t i = tid; i < n * (D / 8); i += KA_THREADS)
      reinterpret_cast<uint4 *>(p.out + row0 * D)[i] = make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (size_t i = tid; i < n; i += KA_THREADS) p.lse[row0 + i] = -INFINITY;
  }

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
  constexpr int CPR = D / 16, STEP = KA_THREADS / CPR, NC = KT / STEP, NG = KT / 16;
  const int ch = tid % CPR, key0 = tid / CPR;
  const uint32_t pool_step = (uint32_t)(H * p.c.page * D);
  // Offsets in a stage (K, then V): the copy's first chunk; the first key of
  // this warp's 16-key groups, spans of 64 dims of either parity (the swizzle of
  // a key is the same 8 keys on); the first two keys of this lane's PV step.
  const uint32_t copy_at = ka_chunk<D>(key0, ch);
  const uint32_t k_at0 = ka_chunk<D>(16 * warp * MW + g, c), k_at1 = k_at0 ^ 64;
  const int v_ch = D == 64 ? warp : 2 * T::ND * warp + (g >> 2);
  const uint32_t v_in = D == 64 ? g * 2 : (g & 3) * 4;
  const uint32_t v_at0 = KA_TILE + ka_chunk<D>(2 * c, v_ch) + v_in;
  const uint32_t v_at1 = KA_TILE + ka_chunk<D>(2 * c + 1, v_ch) + v_in;
  // (32 dims on, two chunks: the swizzle flips bits 1 and 2 of the chunk number)
  const uint32_t v_next0 = D == 256 ? KA_TILE + ka_chunk<D>(2 * c, v_ch + 2) + v_in - v_at0 : 0;
  const uint32_t v_next1 =
      D == 256 ? KA_TILE + ka_chunk<D>(2 * c + 1, v_ch + 2) + v_in - v_at1 : 0;

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
    const unsigned long long u0 = w0 - t0;  // the unit's first tile
    w0 += t1 - t0;
    const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
    const int8_t *kbase = p.c.k_codes + (size_t)h * p.c.page * D + ch * 16;
    const int8_t *vbase = p.c.v_codes + (size_t)h * p.c.page * D + ch * 16;

    // Table entry of the 16-key group lane % NG of a tile (-1: past the last key).
    // Rows without a page read page 0 and get no weight.
    auto group_entry = [&](int t) {
      const int key = t * KT + (lane % NG) * 16;
      return t < t1 && key < kend ? kv8_page_load(table, p.c.max_pages, key >> p.shift) : -1;
    };
    // K scale of the group (-1 masks it) and V scale
    auto group_scales = [&](int entry, float &ks, float &vs) {
      const bool there = (unsigned)entry < (unsigned)p.c.pages;
      ks = there ? __ldg(p.c.k_scales + (size_t)entry * H + h) : -1.f;
      vs = there ? __ldg(p.c.v_scales + (size_t)entry * H + h) : 0.f;
    };
    auto issue = [&](int t, int stage, int entry) {
      int id = entry;
      if ((unsigned)entry >= (unsigned)p.c.pages) {
        if (t * KT + (lane % NG) * 16 < kend) flag_status(p.status, VB_STATUS_BOUNDS);
        id = 0;
      }
      uint8_t *dst = smem + stage * (2 * KA_TILE) + copy_at;
      const int in_page = (t * KT) & (p.c.page - 1);  // 0 unless a page is longer than a tile
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int kl = key0 + i * STEP;
        const uint32_t pg = (uint32_t)__shfl_sync(0xffffffffu, id, kl >> 4);
        const unsigned long long at = (unsigned long long)pg * pool_step +
                                      (uint32_t)((in_page + (kl & (p.c.page - 1))) * D);
        cp_async16(dst + i * STEP * D, kbase + at);
        cp_async16(dst + KA_TILE + i * STEP * D, vbase + at);
      }
    };
    // entries of the tiles t + 1 (id1) and t + 2 (id2) at the start of tile t
    int id1 = group_entry(t0);
    float ks_l, vs_l;
    group_scales(id1, ks_l, vs_l);
    issue(t0, 0, id1);
    cp_async_commit();
    id1 = group_entry(t0 + 1);
    int id2 = group_entry(t0 + 2);
    if (tid < 2) s_move[tid] = 0;

    // ---- queries, in the order of the B fragments: D / 8 lanes per row
    {
      constexpr int LPR = D / 8, PASS = KA_THREADS / LPR, NP = (ROWS + PASS - 1) / PASS;
      const int c8 = tid % LPR;
      uint4 w[NP];
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int r = tid / LPR + k * PASS, i = p.row_of(r), hr = r - i * p.rep;
        w[k] = make_uint4(0, 0, 0, 0);
        if (r < rows && i < sp.q_len)
          w[k] = kv8_load8(p.q + b * p.qb + (int64_t)(h * p.rep + hr) * p.qh +
                               (int64_t)i * p.ql + c8 * 8,
                           p.vec);
      }
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int r = tid / LPR + k * PASS;
        const float pw = kv8_q_scale<LPR>(w[k]);
        if (r >= ROWS) continue;  // (8 rows of 64: half of the threads)
        if (c8 == 0) s_fac[r] = p.scale_log2 / pw;
        // dims 8 c8 .. + 7: d = 64 span + 16 c + 4 step + y; two steps of lane (row, c)
        const int fl = (r & 7) * 4 + ((c8 & 7) >> 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int step = (c8 >> 3) * 4 + (c8 & 1) * 2 + j;
          *reinterpret_cast<uint2 *>(
              s_q + (((r >> 3) * (D / 32) + (step >> 1)) * 32 + fl) * 4 + (step & 1) * 2) =
              j ? make_uint2(w[k].z, w[k].w) : make_uint2(w[k].x, w[k].y);
        }
      }
    }

    // row 8 n + 2 c + u of this lane
    int vis[NR][2];
    float fac[NR][2], m[NR][2], l[NR][2];
    float o[NM][NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = n * 8 + 2 * c + u;
        vis[n][u] = r < rows ? sp.visible(p.row_of(r)) : 0;
        m[n][u] = -INFINITY;
        l[n][u] = 0.f;
      }
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[i][n][u] = 0.f;
    float vref = 0.f, vinv = 0.f;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) fac[n][u] = s_fac[n * 8 + 2 * c + u];

    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      cp_async_wait<0>();
      __syncthreads();  // tile t is in; every warp is done with tile t - 1
      if (t + 1 < t1) issue(t + 1, stage ^ 1, id1);
      cp_async_commit();
      if (tid == 0) s_move[(t + 1) & 1] = 0;
      float ks_n, vs_n;  // of tile t + 1
      group_scales(id1, ks_n, vs_n);
      id1 = id2;
      id2 = group_entry(t + 3);
      const uint8_t *st = smem + stage * (2 * KA_TILE);
      stage ^= 1;

      // ---- S^T = K q^T
      float acc[MW][NR][4];
#pragma unroll
      for (int j = 0; j < MW; ++j)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[j][n][u] = 0.f;
#pragma unroll
      for (int s = 0; s < D / 64; ++s) {
#pragma unroll
        for (int j = 0; j < MW; ++j) {
          const uint8_t *kp = st + ((s & 1) ? k_at1 : k_at0) + 16 * j * D + (s >> 1) * 128;
          const uint4 lo = *reinterpret_cast<const uint4 *>(kp);
          const uint4 hi = *reinterpret_cast<const uint4 *>(kp + 8 * D);
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const uint32_t w = (r4 == 0 ? lo.x : r4 == 1 ? lo.y : r4 == 2 ? lo.z : lo.w) ^ 0x80808080u;
            const uint32_t v = (r4 == 0 ? hi.x : r4 == 1 ? hi.y : r4 == 2 ? hi.z : hi.w) ^ 0x80808080u;
            const uint4 a = make_uint4(h2_codes(__byte_perm(w, 0x64646464u, 0x4140)),
                                       h2_codes(__byte_perm(v, 0x64646464u, 0x4140)),
                                       h2_codes(__byte_perm(w, 0x64646464u, 0x4342)),
                                       h2_codes(__byte_perm(v, 0x64646464u, 0x4342)));
            const int step = s * 4 + r4;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              const uint2 bq = *reinterpret_cast<const uint2 *>(
                  s_q + ((n * (D / 32) + (step >> 1)) * 32 + lane) * 4 + (step & 1) * 2);
              mma_f16(acc[j][n], a, bq.x, bq.y);
            }
          }
        }
      }

      // ---- scores; does a row's maximum or the V scale have to move?
      float vmax = vs_l;
#pragma unroll
      for (int o2 = NG / 2; o2 > 0; o2 >>= 1)
        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o2));
      float vs[MW], lim[NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) lim[n][u] = __fadd_rd(m[n][u], KA_SHIFT + KA_MOVE);
      bool over = vmax > vref;
#pragma unroll
      for (int j = 0; j < MW; ++j) {
        const int grp = warp * MW + j;
        const float ks = __shfl_sync(0xffffffffu, ks_l, grp);
        vs[j] = __shfl_sync(0xffffffffu, vs_l, grp);
        const int key = ks < 0.f ? 0x7fffffff - 64 : t * KT + grp * 16 + g;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float z = acc[j][n][u] * (fac[n][u & 1] * ks);
            acc[j][n][u] = key + (u >> 1) * 8 < vis[n][u & 1] ? z : -INFINITY;
            over |= acc[j][n][u] > lim[n][u & 1];
          }
      }
      ks_l = ks_n;
      vs_l = vs_n;
      if (over) s_move[t & 1] = 1;

      // ---- weights as B fragments of the second product: [key][8 rows] f16
      float add[NR][2];
      auto weights = [&]() {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float sub0 = m[n][0] == -INFINITY ? 0.f : m[n][0];
          const float sub1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
          add[n][0] = add[n][1] = 0.f;
#pragma unroll
          for (int j = 0; j < MW; ++j) {
            const float f = vs[j] * vinv;
            const int key = (warp * MW + j) * 16 + g;
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // keys g and g + 8
              const float e0 = kv8_ex2(acc[j][n][2 * u] - sub0);
              const float e1 = kv8_ex2(acc[j][n][2 * u + 1] - sub1);
              add[n][0] += e0;
              add[n][1] += e1;
              *reinterpret_cast<uint32_t *>(s_p + (n * KT + key + 8 * u) * 16 + c * 4) =
                  pack_h2(e0 * f, e1 * f);
            }
          }
        }
      };
      weights();
      __syncthreads();
      if (s_move[t & 1]) {  // (every warp alike) take the new maximum and scale
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x = -INFINITY;
#pragma unroll
            for (int j = 0; j < MW; ++j) x = fmaxf(x, fmaxf(acc[j][n][u], acc[j][n][2 + u]));
#pragma unroll
            for (int o2 = 4; o2 < 32; o2 <<= 1)
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o2));
            if (g == 0) s_max[warp][n * 8 + 2 * c + u] = x;
          }
        __syncthreads();
        const float vnew = fmaxf(vref, vmax);
        vinv = vnew >= 1.1754944e-38f ? __frcp_rn(vnew) : 0.f;  // (below 2^-126: read as 0)
        const float vold = vref * vinv;
        vref = vnew;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int r = n * 8 + 2 * c + u;
            const float top = fmaxf(fmaxf(s_max[0][r], s_max[1][r]),
                                    fmaxf(s_max[2][r], s_max[3][r]));
            const float mn = fmaxf(__fadd_ru(top, -KA_SHIFT), m[n][u]);
            const float alpha = mn == -INFINITY ? 0.f : kv8_ex2(m[n][u] - mn);
            m[n][u] = mn;
            l[n][u] *= alpha;
#pragma unroll
            for (int i = 0; i < NM; ++i) {
              o[i][n][u] *= alpha * vold;
              o[i][n][2 + u] *= alpha * vold;
            }
          }
        weights();
        __syncthreads();
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        l[n][0] += add[n][0];
        l[n][1] += add[n][1];
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int s = 0; s < KT / 16; ++s) {
        uint32_t bp[NR][2];
#pragma unroll
        for (int n = 0; n < NR; ++n)
          ldsm_x2_trans(bp[n][0], bp[n][1], s_p + (n * KT + s * 16 + (lane & 15)) * 16);
#pragma unroll
        for (int d = 0; d < T::ND; ++d) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t *vp = st + ((i & 1) ? v_at1 + d * v_next1 : v_at0 + d * v_next0) +
                                (s * 16 + (i >> 1) * 8) * D;
            w[i] = (D == 64 ? (uint32_t)*reinterpret_cast<const uint16_t *>(vp)
                            : *reinterpret_cast<const uint32_t *>(vp)) ^ 0x80808080u;
          }
          const uint32_t x0 = __byte_perm(w[0], w[1], 0x5140), x1 = __byte_perm(w[0], w[1], 0x7362);
          const uint32_t y0 = __byte_perm(w[2], w[3], 0x5140), y1 = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
          for (int i = 0; i < (D == 64 ? 1 : 2); ++i) {  // dims 4 g + 2 i, + 1
            const uint32_t x = i ? x1 : x0, y = i ? y1 : y0;
            const uint4 a = make_uint4(h2_codes(__byte_perm(x, 0x64646464u, 0x4140)),
                                       h2_codes(__byte_perm(x, 0x64646464u, 0x4342)),
                                       h2_codes(__byte_perm(y, 0x64646464u, 0x4140)),
                                       h2_codes(__byte_perm(y, 0x64646464u, 0x4342)));
#pragma unroll
            for (int n = 0; n < NR; ++n) mma_f16(o[2 * d + i][n], a, bp[n][0], bp[n][1]);
          }
        }
      }
    }

    // ---- l over the lanes of a row and the warps
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x = l[n][u];
#pragma unroll
        for (int o2 = 4; o2 < 32; o2 <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o2);
        if (g == 0) s_l[warp][n * 8 + 2 * c + u] = x;
      }
    __syncthreads();  // (and the ring, s_q and s_p are free for the next unit)
    const bool whole = t0 == 0 && t1 == tiles;
    const size_t slot = (size_t)blockIdx.x * 2 + (t0 == 0);
    constexpr int DL = D == 64 ? 2 : 4;  // consecutive dims of this lane per group
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = n * 8 + 2 * c + u;
        if (r >= rows) continue;
        const float ls = (s_l[0][r] + s_l[1][r]) + (s_l[2][r] + s_l[3][r]);
        const int i = p.row_of(r);
        const size_t row = ((size_t)b * p.Hq + h * p.rep + r - i * p.rep) * p.L + i;
        const float mul = !whole ? vref : ls == 0.f ? 0.f : vref / ls;  // 0: sees no key
        if (warp == 0 && g == 0) {
          if (!whole)
            p.ml_part[slot * ROWS + r] = make_float2(m[n][u], ls);
          else if (p.lse)
            p.lse[row] = ls == 0.f ? -INFINITY
                                   : (m[n][u] + log2f(ls)) * 0.69314718055994531f;
        }
#pragma unroll
        for (int d = 0; d < T::ND; ++d) {
          float f[4];
#pragma unroll
          for (int k = 0; k < DL; ++k) f[k] = o[2 * d + (k >> 1)][n][(k & 1) * 2 + u] * mul;
          const int dim = warp * T::DW + d * 32 + g * DL;
          if (!whole) {
            float *dst = p.o_part + (slot * ROWS + r) * D + dim;
            if constexpr (DL == 4)
              *reinterpret_cast<float4 *>(dst) = make_float4(f[0], f[1], f[2], f[3]);
            else
              *reinterpret_cast<float2 *>(dst) = make_float2(f[0], f[1]);
          } else {
            uint16_t *dst = p.out + row * D + dim;
            if constexpr (DL == 4)
              *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]));
            else
              *reinterpret_cast<uint32_t *>(dst) = pack_bf2(f[0], f[1]);
          }
        }
      }
    // the CTAs that share the unit: s_share[1] from s_share[0] on
    if (!whole && p.wide) {
      if (t0 == 0 && tid == 0)
        p.units[b * H + h] =
            make_int2(blockIdx.x, (int)(deal.owner(u0 + tiles - 1) - blockIdx.x) + 1);
    } else if (!whole) {  // the last of them joins the partial results
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const uint32_t c0 = t0 == 0 ? blockIdx.x : deal.owner(u0);
        const uint32_t n = deal.owner(u0 + tiles - 1) - c0 + 1;
        uint32_t *ticket = p.tickets + (b * H + h);
        const bool last = atomicAdd(ticket, 1u) == n - 1;
        if (last) *ticket = 0;
        s_share[0] = (int)c0;
        s_share[1] = last ? (int)n : 0;
      }
      __syncthreads();
      const int n = s_share[1];
      if (n > 0) {
        __threadfence();
        const size_t c0 = s_share[0];
        // the first CTA's slot 1, then slot 0 of the following ones
        auto at = [&](int s) { return ((c0 + s) * 2 + (s == 0)) * ROWS; };
        // a row's weights 2^(m_s - M) (in the ring) and its M and l
        float *wgt = reinterpret_cast<float *>(smem);  // [n][ROWS]
#pragma unroll 2
        for (int r = warp; r < rows; r += 4) {
          const float2 first = lane < n ? __ldcg(p.ml_part + at(lane) + r)
                                        : make_float2(-INFINITY, 0.f);
          float M = first.x, ls = 0.f;
          for (int s = lane + 32; s < n; s += 32) M = fmaxf(M, __ldcg(p.ml_part + at(s) + r).x);
#pragma unroll
          for (int o2 = 16; o2 > 0; o2 >>= 1)
            M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o2));
          for (int s = lane; s < n; s += 32) {
            const float2 ml = s == lane ? first : __ldcg(p.ml_part + at(s) + r);
            const float w = ml.x == -INFINITY ? 0.f : kv8_ex2(ml.x - M);
            wgt[s * ROWS + r] = w;
            ls = fmaf(w, ml.y, ls);
          }
#pragma unroll
          for (int o2 = 16; o2 > 0; o2 >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o2);
          if (lane == 0) {
            s_max[0][r] = M;
            s_l[0][r] = ls;
          }
        }
        __syncthreads();
        constexpr int RT = KA_THREADS * 4 / D, IT = (ROWS + RT - 1) / RT;  // rows at a time, turns
        const int d4 = tid % (D / 4), r0 = tid / (D / 4);
        constexpr int IG = IT < 4 ? IT : 4;  // rows of this thread at a time
#pragma unroll 1
        for (int i0 = 0; i0 < IT; i0 += IG) {
          float4 a[IG];
#pragma unroll
          for (int i = 0; i < IG; ++i) a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 6
          for (int s = 0; s < n; ++s) {
            float4 x[IG];
#pragma unroll
            for (int i = 0; i < IG; ++i) {
              const int r = min(r0 + (i0 + i) * RT, rows - 1);
              x[i] = __ldcg(reinterpret_cast<const float4 *>(p.o_part + (at(s) + r) * D) + d4);
            }
#pragma unroll
            for (int i = 0; i < IG; ++i) {
              const int r = min(r0 + (i0 + i) * RT, rows - 1);
              const float w = wgt[s * ROWS + r];
              a[i].x = fmaf(w, x[i].x, a[i].x);
              a[i].y = fmaf(w, x[i].y, a[i].y);
              a[i].z = fmaf(w, x[i].z, a[i].z);
              a[i].w = fmaf(w, x[i].w, a[i].w);
            }
          }
#pragma unroll
          for (int i = 0; i < IG; ++i) {
            const int r = r0 + (i0 + i) * RT;
            if (r < rows) kv8_finish(p, D, b, h, r, d4, s_max[0][r], s_l[0][r], a[i]);
          }
        }
      }
    } else if (p.wide && tid == 0) {
      p.units[b * H + h] = make_int2(blockIdx.x, 1);
    }
    if (w0 < w1) __syncthreads();  // s_l has been read
  }
}

// ------------------------------------------------------------------- combine
constexpr int KC_THREADS = 256;
constexpr int KC_FIRST = 8;  // partial results a thread reads ahead
constexpr int KC_MAX = 512;  // most partial results of one row

// The prefill kernel's row tiles with few key ranges each: a thread joins four
// dims of one row.
template <int D>
__global__ void __launch_bounds__(KC_THREADS) kv8_combine_kernel(Kv8AttnParams p, int tile_rows) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int RPC = KC_THREADS * 4 / D;  // rows per CTA
  const int rows = p.L * p.rep, groups = (rows + RPC - 1) / RPC;
  const int bh = blockIdx.x / groups, R = blockIdx.x % groups * RPC + threadIdx.x / (D / 4);
  const int b = bh / p.c.kv_heads, h = bh % p.c.kv_heads;
  if (R >= rows) return;
  const size_t first = ((size_t)bh * p.row_tiles + R / tile_rows) * p.splits;
  const int r = R % tile_rows;
  kv8_join<D>(p, b, h, R, threadIdx.x % (D / 4), p.splits,
              [&](int s) { return (first + s) * tile_rows + r; });
}

// Where a row's partial results are, for the wide kernel: kv8_attn_kernel's
// units (`units` not null): slot 1 of the first CTA that shares the unit, slot 0
// of the following ones; n = 1: finished by that CTA, n = 0: no keys. The
// prefill kernel: `splits` per row tile.
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
    q.n = kv8_tiles<KA_TILE / D>(p, b, false) > 0 ? u.y : 0;
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

// For many partial results per row: a CTA takes 32 dims of one row, 8 threads
// per partial result and 32 of them at a time, so that all loads are in flight
// at once.
template <int D>
__global__ void __launch_bounds__(KC_THREADS) kv8_combine_wide_kernel(Kv8AttnParams p,
                                                                      int tile_rows) {
  __shared__ float s_w[KC_MAX];
  __shared__ float4 s_acc[KC_THREADS / 32][8];
  __shared__ float s_red[KC_THREADS / 32], s_ls[KC_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rows = p.L * p.rep;
  const int R = blockIdx.x % rows, bh = blockIdx.x / rows;
  const int b = bh / p.c.kv_heads, h = bh % p.c.kv_heads;
  const int d4 = blockIdx.y * 8 + (tid & 7), grp = tid >> 3, r = R % tile_rows;
  const Kv8Parts q = kv8_parts<D>(p, bh, b, R / tile_rows);
  if (p.units && q.n <= 1) return;
  auto part = [&](int s) {
    return __ldcg(reinterpret_cast<const float4 *>(p.o_part + (q.at(s) * tile_rows + r) * D) + d4);
  };
  // the first 256 are on their way while the weights are made (a result without
  // keys has none written: it is read, but not used)
  float4 x[KC_FIRST];
#pragma unroll
  for (int k = 0; k < KC_FIRST; ++k) {
    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp + 32 * k < q.n) x[k] = part(grp + 32 * k);
  }
  float M = -INFINITY, ls = 0.f;
  float2 ml[KC_MAX / KC_THREADS];
#pragma unroll
  for (int k = 0; k < KC_MAX / KC_THREADS; ++k) {
    const int s = tid + k * KC_THREADS;
    ml[k] = s < q.n ? __ldcg(p.ml_part + q.at(s) * tile_rows + r) : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[k].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KC_THREADS / 32; ++w) M = fmaxf(M, s_red[w]);
#pragma unroll
  for (int k = 0; k < KC_MAX / KC_THREADS; ++k) {
    const float wgt = ml[k].x == -INFINITY ? 0.f : kv8_ex2(ml[k].x - M);
    s_w[tid + k * KC_THREADS] = wgt;
    ls = fmaf(wgt, ml[k].y, ls);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
  if ((tid & 31) == 0) s_ls[tid >> 5] = ls;
  __syncthreads();
  ls = 0.f;
#pragma unroll
  for (int w = 0; w < KC_THREADS / 32; ++w) ls += s_ls[w];
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float w, const float4 &y) {
    if (w > 0.f) {
      a.x = fmaf(w, y.x, a.x); a.y = fmaf(w, y.y, a.y);
      a.z = fmaf(w, y.z, a.z); a.w = fmaf(w, y.w, a.w);
    }
  };
#pragma unroll
  for (int k = 0; k < KC_FIRST; ++k)
    if (grp + 32 * k < q.n) add(s_w[grp + 32 * k], x[k]);
#pragma unroll 8
  for (int s = grp + 32 * KC_FIRST; s < q.n; s += 32) {
    const float w = s_w[s];
    if (w > 0.f) add(w, part(s));
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    a.x += __shfl_xor_sync(0xffffffffu, a.x, o); a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
    a.z += __shfl_xor_sync(0xffffffffu, a.z, o); a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
  if ((tid & 31) < 8) s_acc[tid >> 5][tid & 7] = a;
  __syncthreads();
  if (tid >= 8) return;
#pragma unroll
  for (int k = 1; k < KC_THREADS / 32; ++k) {
    const float4 y = s_acc[k][tid];
    a.x += y.x; a.y += y.y; a.z += y.z; a.w += y.w;
  }
  kv8_finish(p, D, b, h, R, d4, M, ls, a);
}

// ---------------------------------------------------------------------- plan
struct Kv8Plan {
  int tile_rows, row_tiles, splits, ctas;
  bool tensor;
  size_t parts, unit_bytes, bytes;  // partial results (tile_rows rows each), workspace
  bool wide;            // many partial results per row
};

// Key ranges per row tile for `base` row tiles of up to `tiles` key tiles. Time in
// key tiles: waves of 74 pairs of CTAs, each with its keys and 3 for its start and
// end, and where there are several ranges their joining. Ranges have to promise a
// tenth: 80 row tiles over 16,384 keys of 256 take 374 us in ranges and 452 whole, 8
// over 4,096 27 and 61, 38 over 131,072 keys of 128 780 and 1,594, but 104 over 3,000
// keys of 128 82 in two ranges and 70 whole (promise: 1 %).
int kv8_ranges(long long base, long long tiles) {
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= 74 && s <= tiles && (s == 1 || base * s <= 8 * 74); ++s) {
    const double waves = (double)((base * s + 73) / 74);
    const double joined = s > 1 ? 2 + base * s / 32. : 0;
    const double cost = waves * (3 + (double)((tiles + s - 1) / s)) + joined;
    if (cost < least * (best == 1 && s > 1 ? 0.9 : 1.)) least = cost, best = s;
  }
  return best;
}

// The plan follows from the table's width (lengths are on the device): the times below
// are of tables as long as their sequences. In a table for 131,072 positions one row
// over 901 keys takes 8.8 us on the device (11.4 in one for 901), 512 rows over 512
// keys of 16/2 heads of 256 49.7 us (18.5), over 8,192 keys 116 (79).
// Up to 32 rows per kv head: kv8_attn_kernel, 8, 16 or 32 rows, its CTAs on
// each of 148 SMs (fewer when the table holds fewer tiles). More rows: the
// tcgen05 kernel, a pair of CTAs per two SMs. (32 rows: 16 sequences of 8,190 keys, 8
// heads of 128, 103 us by the first and 216 by the second; one of 131,072 keys, 2
// heads of 256, 58 and 79.)
Kv8Plan kv8_plan(const VbKv8AttnArgs *a) {
  Kv8Plan pl;
  const long long rows = (long long)a->L * (a->q_heads / a->cache.kv_heads);
  const long long units = (long long)a->cache.batch * a->cache.kv_heads;
  const long long cap = (long long)a->cache.max_pages * a->cache.page;
  pl.tensor = rows > 32;
  if (pl.tensor) {
    pl.tile_rows = kv8_prefill_rows();
    pl.row_tiles = (int)((rows + pl.tile_rows - 1) / pl.tile_rows);
    const long long base = units * pl.row_tiles, tiles = (cap + 127) / 128;
    const int s = kv8_ranges(base, tiles);
    pl.splits = s;
    pl.ctas = 0;
    pl.parts = s == 1 ? 0 : (size_t)(base * s);
  } else {
    pl.tile_rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    pl.row_tiles = pl.splits = 1;
    const long long kt = KA_TILE / a->cache.dim, tiles = units * ((cap + kt - 1) / kt);
    const int full = 148 * (pl.tile_rows == 32 ? Kv8Tile<64, 4>::CTAS : Kv8Tile<64, 1>::CTAS);
    pl.ctas = (int)(tiles < full ? tiles : full);
    pl.parts = (size_t)pl.ctas * 2;
  }
  // Decode: up to 16 units that several CTAs share are joined by the wide kernel, more
  // by the last CTA of each, which then work side by side (wide and last CTA, on the
  // device: heads of 128, 16 rows over 4,000 keys: 2 units 9.6 us and 15.8, 8 12.1 and
  // 17.6, 24 21.3 and 21.9, 48 33.8 and 25.8; heads of 256, 8 rows: 2 9.8 and 21.1, 24
  // 24.6 and 24.2, 48 38.1 and 29.1). Few results are left to the last CTA as well: a
  // second launch costs a call outside a graph 2 us (1 row over 901 keys, 16/2 heads of
  // 256: 8.8 and 12.3 on the device, 17.4 and 15.4 a call; 32 rows always gain, 1,000
  // keys of 64 10.9 and 15.8, and so do many results, 7 rows over 58,182 keys of 64 in
  // 8 units 21.9 and 27.2). Ranges of the prefill kernel: the wide kernel for many
  // of few rows (256 rows 87 us and 93, 1,280 rows 116 and 105, 1,600 rows 115 and 82).
  const bool shared = units <= 16 && pl.ctas > units &&
                      (rows > 16 || pl.ctas > 24 * units ||
                       pl.ctas * rows * a->cache.dim > 40000 * units);
  pl.wide = pl.tensor ? pl.splits > 8 && units * rows <= 512 : shared || units > KA_TICKETS;
  pl.unit_bytes = pl.wide && !pl.tensor ? align_up(units * sizeof(int2), 16) : 0;
  pl.bytes = pl.parts == 0 ? 0
                           : KA_TICKETS * sizeof(uint32_t) + pl.unit_bytes +
                                 pl.parts * pl.tile_rows * (a->cache.dim + 2) * sizeof(float);
  return pl;
}

template <int D, int NR>
int kv8_launch(const Kv8AttnParams &p, int ctas, cudaStream_t s) {
  using T = Kv8Tile<D, NR>;
  static std::atomic<uint64_t> ready{0};
  const int rc = once_per_device(ready, [] {
    const cudaError_t e = cudaFuncSetAttribute(
        kv8_attn_kernel<D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    return e == cudaSuccess ? VB_OK
                            : set_error(VB_ERR_CUDA, "kv8_attn_kernel attributes: %s",
                                        cudaGetErrorString(e));
  });
  if (rc != VB_OK) return rc;
  // Dependent launch for short calls only: started before the kernel ahead has
  // left its SMs, a full grid is placed unevenly (131,072 keys: 49.6 us instead of
  // 37.7; 901 keys: 12.1 us instead of 14.1).
  vb_launch(kv8_attn_kernel<D, NR>, dim3(ctas), dim3(KA_THREADS), T::SMEM, s, ctas <= 148, p);
  return check_launch("kv8_attn_kernel");
}

template <int D>
int kv8_run(const Kv8AttnParams &p, const Kv8Plan &pl, cudaStream_t s) {
  const int rc = pl.tensor ? kv8_prefill_launch(p, s)
                 : pl.tile_rows == 8  ? kv8_launch<D, 1>(p, pl.ctas, s)
                 : pl.tile_rows == 16 ? kv8_launch<D, 2>(p, pl.ctas, s)
                                      : kv8_launch<D, 4>(p, pl.ctas, s);
  if (rc != VB_OK || pl.parts == 0 || (!pl.tensor && !pl.wide)) return rc;
  const unsigned units = p.c.batch * p.c.kv_heads, rows = p.L * p.rep;
  constexpr unsigned RPC = KC_THREADS * 4 / D;
  if (pl.wide)
    vb_launch(kv8_combine_wide_kernel<D>, dim3(units * rows, D / 32), dim3(KC_THREADS), 0, s, true,
              p, pl.tile_rows);
  else
    vb_launch(kv8_combine_kernel<D>, dim3(units * ((rows + RPC - 1) / RPC)), dim3(KC_THREADS), 0, s,
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
  // the tickets lie at the same place in every call: they are zero between calls
  uint8_t *ws = static_cast<uint8_t *>(a->workspace);
  p.tickets = reinterpret_cast<uint32_t *>(ws);
  ws += KA_TICKETS * sizeof(uint32_t);
  p.units = pl.unit_bytes ? reinterpret_cast<int2 *>(ws) : nullptr;
  p.o_part = reinterpret_cast<float *>(ws + pl.unit_bytes);
  p.ml_part = reinterpret_cast<float2 *>(p.o_part + pl.parts * pl.tile_rows * a->cache.dim);
  p.wide = pl.wide;
  cudaStream_t s = as_stream(stream);
  switch (a->cache.dim) {
    case 64: return kv8_run<64>(p, pl, s);
    case 128: return kv8_run<128>(p, pl, s);
    default: return kv8_run<256>(p, pl, s);
  }
}

}  // extern "C"
