// Attention weight that the rows of the paged 8-bit cache receive, added up:
//
//   w_j += sum over query heads of the kv head, rows i that see j, of
//          exp(scale * q_i . k_j - lse_i)
//
// with lse_i from the attention itself, so no row needs another key than j and
// V is not read. The products are those of the attention kernels: codes and
// queries (after a power of two per row) are exact in f16, sums float32, and a
// key's weights are added in one order, whatever the launch.
//
// Up to 32 query rows per kv head (kv8_weigh_kernel, which reads a byte per cached value
// of K): a warp takes 16 keys at a time, brought by cp.async into a ring of its own in
// which every lane finds the 16-byte pieces that it asked for itself, already in the
// order of the fragments of S^T = K q^T (lane (g, c) has 16 consecutive bytes of keys
// g and g + 8, four k-steps), so that nothing in the loop waits for another thread. Rows
// come eight to a fragment.
//
// More rows (kv8_weigh_rows_kernel, a window at a prompt's end or a prompt's chunk;
// tensor-core- and exponential-bound): a pair of CTAs (tcgen05 cta_group::2) takes
// 256 keys at a time, 128 each, as the M rows of the product and 64 to 256 query
// rows as its N columns, so a thread has a key in its TMEM lane and adds its
// weights by itself. Queries are made ready once by a kernel ahead of it.
//
// What bounds it: 32 sequences of up to 8,190 keys, 32/8 heads of 128, take 30 us for 128
// MB (4.3 TB/s, a copy 19.6): neither HBM nor the issue slots are more than half used
// (five instructions turn four codes into f16); warps wait for their keys, and each of the
// short CTAs for its page numbers and queries first; one sequence of 901 keys costs the launch, 3.5.
// 64 rows of 16/2 heads of 256 over 32,768 keys take 29 us (products alone 10.4): two
// chunks of 256 rows over three or four tiles a pair, 1.8 us each, 4 for the queries and 8
// to begin and end; over 131,072 keys a tile of 256 x 256 takes 2.4 us, of which the
// exponentials fill their pipe for 1.1.
#include "kv8_pair.cuh"

namespace vb {
namespace {

struct Kv8WeighParams {
  Kv8AttnParams a;           // out, lse (written) and workspace are not used
  const float *lse;
  const int32_t *fresh, *seen;  // new rows at the end (null: the query rows), tokens so far
  float *weights;
  int32_t *positions;
  int room, groups;          // groups: 16-key groups of a warp
  // of kv8_weigh_rows_kernel
  uint16_t *q16;             // [batch, kv heads, padded rows, dim]: f16 queries
  float2 *row;               // their score factor, log2 sum (+inf: does not count)
  int padded, ranges;        // rows, key ranges of a (sequence, head)
};

// Keys of sequence b, and the first of its new rows; false: left out.
struct Kv8WeighSpan {
  Kv8Span sp;
  int fresh;
};
__device__ __forceinline__ bool wg_span(const Kv8WeighParams &w, int b, bool flag, Kv8WeighSpan &s) {
  s.sp = kv8_span(w.a, b, flag);
  int32_t *status = flag ? w.a.status : nullptr;
  if (s.sp.keys > w.room) {
    flag_status(status, VB_STATUS_BOUNDS);
    return false;
  }
  s.fresh = s.sp.keys - (w.fresh ? kv8_rows(w.fresh, b, s.sp.keys, status)
                                 : min(s.sp.q_len, s.sp.keys));
  return true;
}
// Adds a key's sum; `first`: the call's first sum of it, with which a new row begins.
__device__ __forceinline__ void wg_add(const Kv8WeighParams &w, const Kv8WeighSpan &s, int b,
                                       size_t at, int key, float sum, bool first, float old) {
  const bool is_new = first && key >= s.fresh;
  if (is_new || sum != 0.f) w.weights[at + key] = (is_new ? 0.f : old) + sum;
  if (is_new && w.positions) w.positions[at + key] = w.seen[b] - (s.sp.keys - key);
}

// ------------------------------------------------------------ few query rows
constexpr int WG_THREADS = 128;
constexpr int WG_WARPS = WG_THREADS / 32;
// Stages of 16 keys in a warp's ring: as little in flight per warp as still hides its own
// computing, so that more warps fit (heads of 128, 3, 4 and 6 stages: 31, 34 and 40 us;
// of 256, 2 and 3: 17 and 22).
template <int D>
constexpr int wg_stages() { return D == 64 ? 3 : 2; }

__device__ __forceinline__ void wg_mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

template <int D, int NR>  // NR groups of 8 query rows
__global__ void __launch_bounds__(WG_THREADS) kv8_weigh_kernel(const __grid_constant__ Kv8WeighParams w) {
  const Kv8AttnParams &p = w.a;
  constexpr int ROWS = 8 * NR, PIECES = D / 32, STAGES = wg_stages<D>();
  extern __shared__ __align__(16) uint8_t ring[];  // [warp][stage][piece][lane][16]
  __shared__ uint32_t s_q[NR * D * 4];             // [8 rows][D/32][32 lanes][4]
  __shared__ float2 s_row[ROWS];                   // score factor, log2 sum
  __shared__ int s_vis[ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int H = p.c.kv_heads, b = blockIdx.z, h = blockIdx.y;
  Kv8WeighSpan s;
  if (!wg_span(w, b, blockIdx.x == 0 && h == 0 && tid == 0, s)) return;
  const int keys = s.sp.keys, key_first = blockIdx.x * (WG_WARPS * 16) * w.groups;
  if (key_first >= keys) return;
  const int rows = s.sp.q_len * p.rep;
  const size_t at0 = ((size_t)b * H + h) * w.room, page_bytes = (size_t)p.c.page * D;
  auto first_key = [&](int it) { return key_first + (it * WG_WARPS + warp) * 16; };
  // page and K scale (-1: no such page) of the group that this lane looks up
  int id = -1;
  float ks_l = -1.f;
  if (lane < w.groups && first_key(lane) < keys) {
    id = kv8_page(p.c.page_table + (size_t)b * p.c.max_pages, p.c.max_pages, p.c.pages,
                  first_key(lane) >> p.shift, p.status);
    if (id >= 0) ks_l = __ldcg(p.c.k_scales + (size_t)id * H + h);
  }
  uint8_t *mine = ring + (warp * STAGES * PIECES * 32 + lane) * 16;
  auto issue = [&](int it) {
    const int pg = max(0, __shfl_sync(0xffffffffu, id, it & 31));
    if (it < w.groups && first_key(it) < keys) {
      const int8_t *k = p.c.k_codes + ((size_t)pg * H + h) * page_bytes +
                        (size_t)((first_key(it) & (p.c.page - 1)) + g) * D + c * 16;
      uint8_t *dst = mine + it % STAGES * (PIECES * 512);
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        cp_async16(dst + 2 * x * 512, k + x * 64);
        cp_async16(dst + (2 * x + 1) * 512, k + x * 64 + 8 * D);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int it = 0; it < STAGES - 1; ++it) issue(it);

  // ---- queries in the order of the B fragments: D / 8 lanes per row
  {
    constexpr int LPR = D / 8, PASS = WG_THREADS / LPR, NP = (ROWS + PASS - 1) / PASS;
    const int c8 = tid % LPR;
    uint4 v[NP];
    float l[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int r = tid / LPR + k * PASS, i = p.row_of(r), hq = h * p.rep + r - i * p.rep;
      v[k] = make_uint4(0, 0, 0, 0);
      l[k] = -INFINITY;
      if (r < rows) {
        v[k] = kv8_load8(p.q + b * p.qb + (int64_t)hq * p.qh + (int64_t)i * p.ql + c8 * 8, p.vec);
        l[k] = w.lse[((size_t)b * p.Hq + hq) * p.L + i];
      }
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int r = tid / LPR + k * PASS;
      const float pw = kv8_q_scale<LPR>(v[k]);
      if (r >= ROWS) continue;  // (8 rows of 64: half of the threads)
      if (c8 == 0) {
        const bool counts = fabsf(l[k]) <= 3.4028235e38f;
        if (!counts && l[k] != -INFINITY && key_first == 0) flag_status(p.status, VB_STATUS_NONFINITE);
        s_row[r] = make_float2(p.scale_log2 / pw, l[k] * 1.4426950408889634f);
        s_vis[r] = counts ? s.sp.visible(p.row_of(r)) : 0;
      }
      const int fl = (r & 7) * 4 + ((c8 & 7) >> 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int step = (c8 >> 3) * 4 + (c8 & 1) * 2 + j;
        *reinterpret_cast<uint2 *>(
            s_q + (((r >> 3) * (D / 32) + (step >> 1)) * 32 + fl) * 4 + (step & 1) * 2) =
            j ? make_uint2(v[k].z, v[k].w) : make_uint2(v[k].x, v[k].y);
      }
    }
  }
  __syncthreads();
  // the fragments of eight rows stay in registers
  constexpr bool HELD = NR == 1;
  uint2 held[HELD ? D / 16 : 1];
  auto fragment = [&](int n, int step) {
    return *reinterpret_cast<const uint2 *>(
        s_q + ((n * (D / 32) + (step >> 1)) * 32 + lane) * 4 + (step & 1) * 2);
  };
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) held[k] = fragment(0, k);
  }
  float2 row[NR][2];
  int vis[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      row[n][u] = s_row[n * 8 + 2 * c + u];
      vis[n][u] = s_vis[n * 8 + 2 * c + u];
    }

  for (int it = 0; it < w.groups; ++it) {
    const int key0 = first_key(it);
    if (key0 >= keys) break;
    const int key = key0 + g + 8 * c;  // (c < 2) the key that this lane adds to
    float old = 0.f;
    if (c < 2 && key < keys) old = w.weights[at0 + key];
    issue(it + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    const uint8_t *st = mine + it % STAGES * (PIECES * 512);
    const float ks = __shfl_sync(0xffffffffu, ks_l, it & 31);
    float acc[NR][2][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int u = 0; u < 8; ++u) acc[n][u >> 2][u & 3] = 0.f;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
      const uint4 lo = *reinterpret_cast<const uint4 *>(st + 2 * x * 512);
      const uint4 hi = *reinterpret_cast<const uint4 *>(st + (2 * x + 1) * 512);
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const uint32_t y = (r4 == 0 ? lo.x : r4 == 1 ? lo.y : r4 == 2 ? lo.z : lo.w) ^ 0x80808080u;
        const uint32_t z = (r4 == 0 ? hi.x : r4 == 1 ? hi.y : r4 == 2 ? hi.z : hi.w) ^ 0x80808080u;
        const uint4 a = make_uint4(h2_codes(__byte_perm(y, 0x64646464u, 0x4140)),
                                   h2_codes(__byte_perm(z, 0x64646464u, 0x4140)),
                                   h2_codes(__byte_perm(y, 0x64646464u, 0x4342)),
                                   h2_codes(__byte_perm(z, 0x64646464u, 0x4342)));
        const int step = x * 4 + r4;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const uint2 bq = HELD ? held[HELD ? step : 0] : fragment(n, step);
          wg_mma(acc[n][step & 1], a, bq.x, bq.y);
        }
      }
    }
    float sum0 = 0.f, sum1 = 0.f;  // keys g and g + 8
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {  // rows 8 n + 2 c + u
        const float f = row[n][u].x * ks;
        const float z0 = fmaf(acc[n][0][u] + acc[n][1][u], f, -row[n][u].y);
        const float z1 = fmaf(acc[n][0][2 + u] + acc[n][1][2 + u], f, -row[n][u].y);
        if (key0 + g < vis[n][u]) sum0 += kv8_ex2(z0);
        if (key0 + g + 8 < vis[n][u]) sum1 += kv8_ex2(z1);
      }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      sum0 += __shfl_xor_sync(0xffffffffu, sum0, o);
      sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
    }
    if (c < 2 && key < keys) wg_add(w, s, b, at0, key, ks < 0.f ? 0.f : c ? sum1 : sum0, true, old);
  }
}

// ----------------------------------------------------------- many query rows
constexpr int WR_THREADS = 896;            // a warpgroup issues, two convert, four add
constexpr int WR_KEYS = 256;               // keys of a pair of CTAs
constexpr int WR_COLS = 256;               // query rows at a time
// Registers per thread of the warpgroups; 72 at launch.
constexpr int WR_REGS = 72, WR_R_MMA = 32, WR_R_CONV = 88, WR_R_ADD = 72;
static_assert(WR_R_MMA + 2 * WR_R_CONV + 4 * WR_R_ADD <= 7 * WR_REGS, "register shares");

template <int D>
struct WrShape {
  static constexpr int TILE = 128 * D * 2;                // f16 of 128 keys, or query rows
  static constexpr int K_OFF = TILE;                      // after the queries: two stages
  static constexpr int SMEM = 3 * TILE + 1024;
};

// f16 queries, row after row of a (sequence, kv head), and what turns a product into
// a weight; rows that are not there, or have no finite lse, count for nothing: they are
// zeros, as the product of a NaN, or of an infinity, is not made -inf by any log2 sum.
template <int D>
__global__ void __launch_bounds__(256) kv8_weigh_q_kernel(const __grid_constant__ Kv8WeighParams w) {
  constexpr int LPR = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const Kv8AttnParams &p = w.a;
  const long long at = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c8 = threadIdx.x % LPR, H = p.c.kv_heads;
  const int unit = (int)(at / w.padded), R = (int)(at - (long long)unit * w.padded);
  if (unit >= p.c.batch * H) return;  // (whole rows of lanes; a row's lanes stay together)
  const int b = unit / H, h = unit - b * H, i = p.row_of(R), hq = h * p.rep + R - i * p.rep;
  const Kv8Span sp = kv8_span(p, b, false);
  uint4 v = make_uint4(0, 0, 0, 0);
  float l = -INFINITY;
  if (i < sp.q_len) {
    v = kv8_load8(p.q + b * p.qb + (int64_t)hq * p.qh + (int64_t)i * p.ql + c8 * 8, p.vec);
    l = w.lse[((size_t)b * p.Hq + hq) * p.L + i];
  }
  const bool counts = fabsf(l) <= 3.4028235e38f;
  if (!counts) v = make_uint4(0, 0, 0, 0);
  const float pw = kv8_q_scale<LPR>(v);
  *(reinterpret_cast<uint4 *>(w.q16 + (size_t)at * D) + c8) = v;
  if (c8 == 0) {
    if (!counts && l != -INFINITY) flag_status(p.status, VB_STATUS_NONFINITE);
    // (a factor above 0: times -inf, what a row does not see)
    w.row[at] = make_float2(fmaxf(p.scale_log2 / pw, 1.1754944e-38f),
                            counts ? l * 1.4426950408889634f : INFINITY);
  }
}

// Some of the threads that add meet.
__device__ __forceinline__ void wr_meet(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

struct WrBarriers {
  uint64_t k_full[2], k_empty[2], s_full[2], s_free[2], q_full, drain;
};

template <int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(WR_THREADS, 1)
    kv8_weigh_rows_kernel(const __grid_constant__ Kv8WeighParams w) {
  using S = WrShape<D>;
  const Kv8AttnParams &p = w.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ __align__(8) WrBarriers bar;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float4 s_row[2][WR_COLS / 2];  // of a chunk: factors and log2 sums of two columns
  __shared__ float s_sum[2][2][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
  pdl_launch_dependents();
  pdl_wait();

  // ---- the pair's keys: tiles [t0, t1) of 256
  const int rank = blockIdx.x & 1, H = p.c.kv_heads;
  const int range = (blockIdx.x >> 1) % w.ranges, unit = (blockIdx.x >> 1) / w.ranges;
  const int b = unit / H, h = unit - b * H;
  Kv8WeighSpan s;
  if (!wg_span(w, b, range == 0 && rank == 0 && h == 0 && tid == 0, s)) return;
  const int keys = s.sp.keys, rows = s.sp.q_len * p.rep;
  const size_t at0 = (size_t)unit * w.room;
  if (rows == 0) {  // new rows alone (64 bits: a stride may lead past 31)
    for (long long key = (long long)s.fresh + blockIdx.x % (2 * w.ranges) * WR_THREADS + tid; key < keys;
         key += 2 * w.ranges * WR_THREADS)
      wg_add(w, s, b, at0, (int)key, 0.f, true, 0.f);
    return;
  }
  const int tiles = (keys + WR_KEYS - 1) / WR_KEYS, share = tiles / w.ranges, rest = tiles % w.ranges;
  const int t0 = range * share + min(range, rest), n_tiles = share + (range < rest);
  if (n_tiles == 0) return;  // (both CTAs)
  const int chunks = (rows + WR_COLS - 1) / WR_COLS, steps = chunks * n_tiles;
  // columns of a chunk: up to 256, a multiple of 64
  auto columns = [&](int ch) { return min(WR_COLS, (rows - ch * WR_COLS + 63) & ~63); };

  if (tid == 32) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bar.k_full[i], 2 * 8);   // converter warps of both CTAs
      tc::mbar_init(&bar.k_empty[i], 1);
      tc::mbar_init(&bar.s_full[i], 1);
      tc::mbar_init(&bar.s_free[i], 2 * 8);   // adding warps of both CTAs
    }
    tc::mbar_init(&bar.q_full, 2);  // both CTAs
    tc::mbar_init(&bar.drain, 1);
    s_abort = 0;
    tc::fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tc::smem_u32(&s_tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  kp_cluster_arrive();
  uint32_t tmem = 0;
  auto ready = [&]() {  // barriers and TMEM of both CTAs are there
    tc::tc_fence_before();
    __syncthreads();
    kp_cluster_wait();
    tc::tc_fence_after();
    tmem = s_tmem;
  };
  volatile int *abort = &s_abort;
  const uint32_t sbase = tc::smem_u32(smem);
  // The warp waits for the n-th completion (from 0) of a barrier; false after a wait of
  // this CTA has given up.
  auto wait = [&](uint64_t *m, int n) {
    const bool there = tc::mbar_wait(m, (uint32_t)(n & 1), abort, KP_WAIT_NS);
    if (!there) s_abort = 1;
    return __all_sync(0xffffffffu, there);
  };

  if (wg == 0) {
    // ================================================== tensor-core issuer
    kp_regs_dec<WR_R_MMA>();
    ready();
    if (warp == 0 && rank == 0) {
      const uint32_t one = kp_elect();
      const uint64_t q_desc = tc::smem_desc_sw128(sbase);
      const uint64_t k_desc = tc::smem_desc_sw128(sbase + S::K_OFF);
      bool ok = true;
      for (int n = 0, ch = 0, t = 0; n < steps && ok; ++n) {
        const int st = n & 1;
        if (t == 0) ok = wait(&bar.q_full, ch);
        ok = ok && wait(&bar.k_full[st], n >> 1);
        if (n >= 2) ok = ok && wait(&bar.s_free[st], (n >> 1) - 1);
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t idesc = kp_idesc(columns(ch), false);
        const uint64_t kd = k_desc + st * (S::TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int off = ((kk >> 2) * KP_BLOCK + (kk & 3) * 32) >> 4;
          kp_mma_ss(one, tmem + st * 256, kd + off, q_desc + off, idesc, kk > 0 ? 1u : 0u);
        }
        kp_commit(one, &bar.s_full[st]);
        kp_commit(one, &bar.k_empty[st]);
        if (++t == n_tiles) t = 0, ++ch;
      }
      // nothing of the pair may be in flight when TMEM is freed
      kp_commit(one, &bar.drain);
      if (!tc::mbar_wait(&bar.drain, 0, nullptr, KP_WAIT_NS)) s_abort = 1;
    }
    __syncwarp();
  } else if (wg < 3) {
    // ================================================== converters
    kp_regs_inc<WR_R_CONV>();
    const int ctid = tid - 128;
    constexpr int KC = D / 16, KSTEP = 256 / KC, KN = 128 / KSTEP;
    const int ch = ctid % KC, kkey = ctid / KC;
    const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
    const size_t pool_step = (size_t)H * p.c.page * D;
    const int8_t *kbase = p.c.k_codes + (size_t)h * p.c.page * D + ch * 16;
    // table entry of the 16-key group lane % 8 of this CTA's half of a tile, asked for well
    // before it is looked at; rows without a page (past the last key, or flagged) read
    // page 0: nothing is added to them
    auto entry_of = [&](int t) {
      const int key = t * WR_KEYS + rank * 128 + (lane & 7) * 16;
      return key < keys ? kv8_page_load(table, p.c.max_pages, key >> p.shift) : 0;
    };
    auto page_of = [&](int entry) { return max(0, kv8_page_ok(entry, p.c.pages, p.status)); };
    auto next = [&](int t) { return t + 1 == n_tiles ? 0 : t + 1; };
    uint4 kr[KN];
    auto load = [&](int id) {
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        const int key = kkey + i * KSTEP;  // a tile's half starts on a page boundary
        const int pg = __shfl_sync(0xffffffffu, id, key >> 4);
        kr[i] = __ldcg(reinterpret_cast<const uint4 *>(kbase + pg * pool_step +
                                                       (key & (p.c.page - 1)) * D));
      }
    };
    const int first = entry_of(t0);
    int t = next(0), entry = entry_of(t0 + t);
    load(page_of(first));
    ready();
    for (int n = 0; n < steps; ++n) {
      const int st = n & 1, entry_now = entry;
      t = next(t);
      entry = entry_of(t0 + t);
      if (n >= 2 && !wait(&bar.k_empty[st], (n >> 1) - 1)) break;
      uint8_t *tile = smem + S::K_OFF + st * S::TILE;
#pragma unroll
      for (int i = 0; i < KN; ++i) kp_store_codes(kr[i], tile, KP_BLOCK, kkey + i * KSTEP, ch);
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) kp_arrive_leader(&bar.k_full[st]);
      if (n + 1 < steps) load(page_of(entry_now));
    }
  } else {
    // ================================================== weights, a thread per key
    // Two pairs of warpgroups take the tiles in turn, so that one's exponentials run while
    // the other waits for its products (all four on each tile: 36 us instead of 34 for
    // 256 rows of each of 2 kv heads over 131,072 keys of 64, 47 and 45 for keys of 256).
    kp_regs_dec<WR_R_ADD>();
    const int e = wg - 3, pair = e >> 1, half = e & 1, r = tid & 127;  // half of the columns; a key
    const float2 *row = w.row + (size_t)unit * w.padded;
    const uint16_t *q16 = w.q16 + (size_t)unit * w.padded * D;
    // This CTA's half of a chunk's queries, and the factors of all of its columns, by
    // `threads` threads, this one the `at`-th.
    auto load_q = [&](int ch, int at, int threads) {
      const int rows = columns(ch) / 2, first = ch * WR_COLS + rank * rows;
      for (int x = at; x < rows * (D / 8); x += threads) {
        const int qr = x / (D / 8), c8 = x % (D / 8);
        cp_async16(smem + (c8 >> 3) * KP_BLOCK + kp_sw(qr, c8 & 7),
                   q16 + (size_t)(first + qr) * D + c8 * 8);
      }
      cp_async_commit();
      if (at < 2 * rows) {
        const float2 f = row[ch * WR_COLS + at];
        float *d = reinterpret_cast<float *>(&s_row[ch & 1][at >> 1]) + (at & 1);
        d[0] = f.x;
        d[2] = -f.y;
      }
    };
    auto publish_q = [&](int id, int threads, bool one) {
      cp_async_wait<0>();
      tc::fence_proxy_async_smem();
      wr_meet(id, threads);
      if (one) kp_arrive_leader(&bar.q_full);
    };
    load_q(0, tid - 384, 512);
    // K scale of this thread's key (-1: no such page), a tile ahead, and its table entry
    // another one
    const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
    auto entry_of = [&](int t) {
      const int key = t * WR_KEYS + rank * 128 + r;
      return key < keys ? kv8_page_load(table, p.c.max_pages, key >> p.shift) : -1;
    };
    auto scale_of = [&](int entry) {
      return (unsigned)entry < (unsigned)p.c.pages
                 ? __ldcg(p.c.k_scales + (size_t)entry * H + h) : -1.f;
    };
    auto ahead = [&](int t, int by) { return (t + by) % n_tiles; };
    int t = ahead(0, pair), t_next = ahead(t, 2);
    const int entry_0 = entry_of(t0 + t);
    int entry_n = entry_of(t0 + t_next);
    float ks_n = scale_of(entry_0);
    ready();
    publish_q(1, 512, tid == 384);
    const uint32_t trow = tmem + (((uint32_t)(warp & 3) * 32u) << 16);
    // keys that every query row sees
    const int seen_by_all = s.sp.causal ? max(0, s.sp.off + 1) : keys;
    // After a wait has given up, the tiles are gone through without further ones, as the
    // warpgroups meet in every tile.
    bool ok = true;
    for (int n = pair, ch = 0; n < steps; n += 2) {  // tile t of chunk ch, in S slot n % 2
      // From chunk to chunk the pairs meet: a key's sum goes on where the other may have left
      // it. (Both come here for every chunk, whichever of its tiles they have.)
      for (; ch < n / n_tiles; ++ch) wr_meet(8, 512);
      const int cols = columns(ch), use = n >> 1;
      const float ks = ks_n;
      const bool more = t == n_tiles - 1 && ch + 1 < chunks;
      ks_n = scale_of(entry_n);
      const int key = (t0 + t) * WR_KEYS + rank * 128 + r;
      const bool masked = (t0 + t) * WR_KEYS + rank * 128 + 128 > seen_by_all ||
                          __any_sync(0xffffffffu, ks == 0.f);
      t = t_next;
      t_next = ahead(t, 2);
      entry_n = entry_of(t0 + t_next);
      float old = 0.f;
      if (half == 0 && key < keys) old = w.weights[at0 + key];
      ok = ok && wait(&bar.s_full[pair], use);
      tc::tc_fence_after();
      if (more && ok) load_q(ch + 1, tid - 384 - 256 * pair, 256);  // no product of this chunk is left
      const int first = half * (cols / 2);
      const float4 *tab = s_row[ch & 1] + first / 2;
      // Scale 0: scores of 0 whatever the codes, by products of 0 and a factor above 0, with
      // which a hidden one stays -inf. (No scale stands for 0: a query may undo it.)
      const uint32_t code = ks == 0.f ? 0u : 0xFFFFFFFFu;
      const float kf = ks > 0.f ? ks : 1.f;
      const f2 kk = f2_make(kf, kf);
      const int from = s.sp.causal ? max(0, key - s.sp.off) * p.rep : 0;
      f2 s0 = f2_make(0.f, 0.f), s1 = s0;
#pragma unroll 1
      for (int c0 = 0; c0 < cols / 2; c0 += 32) {
        uint32_t v[32];
        tc::tmem_ld32(trow + pair * 256 + first + c0, v);
        tc::tmem_ld_wait();
        if (masked) {  // query rows from `from` on see this key
          const int hidden = from - (ch * WR_COLS + first + c0);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            v[j] = j < hidden ? 0xFF800000u : v[j] & code;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 x = tab[(c0 + j) / 2], y = tab[(c0 + j) / 2 + 1];
          float z[4];
          f2_split(f2_fma(f2_mul(f2_make(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), kk),
                          f2_make(x.x, x.y), f2_make(x.z, x.w)), z[0], z[1]);
          f2_split(f2_fma(f2_mul(f2_make(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), kk),
                          f2_make(y.x, y.y), f2_make(y.z, y.w)), z[2], z[3]);
          s0 = f2_add(s0, f2_make(kv8_ex2(z[0]), kv8_ex2(z[1])));
          s1 = f2_add(s1, f2_make(kv8_ex2(z[2]), kv8_ex2(z[3])));
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) kp_arrive_leader(&bar.s_free[pair]);
      float a0, a1, a2, a3;
      f2_split(s0, a0, a1);
      f2_split(s1, a2, a3);
      const float sum = (a0 + a1) + (a2 + a3);
      // One warpgroup of the pair adds the sums of both. The other need not wait for it:
      // before it is here with the second tile from now, the first has given back the slot of
      // the next, and so read this one's sums. (Not so after a wait has given up: a second
      // arrival could then complete the barrier without the first, which would wait for good.)
      const int id = 2 + 2 * pair + (use & 1);
      if (half) {
        s_sum[pair][use & 1][r] = sum;
        if (ok) asm volatile("bar.arrive %0, 256;" ::"r"(id) : "memory");
        else wr_meet(id, 256);
      } else {
        wr_meet(id, 256);
        if (ok && key < keys)
          wg_add(w, s, b, at0, key, ks < 0.f ? 0.f : sum + s_sum[pair][use & 1][r], ch == 0, old);
      }
      if (more) publish_q(6 + pair, 256, ok && tid == 384 + 256 * pair);
      if (n + 2 >= steps)
        for (; ch < chunks - 1; ++ch) wr_meet(8, 512);
    }
    if (pair >= steps)
      for (int ch = 0; ch < chunks - 1; ++ch) wr_meet(8, 512);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort) flag_status(p.status, VB_STATUS_TIMEOUT);
  // no product reads the other CTA's operands any more, and all that the leader's
  // products signal has come
  if (warp == 0 && rank == 1) tc::mbar_wait(&bar.drain, 0, nullptr, KP_WAIT_NS);
  // (after a wait gave up, arrivals may be under way that nothing has waited for)
  if (*abort) asm volatile("fence.acq_rel.cluster;" ::: "memory");
  __syncwarp();
  kp_cluster_arrive();
  kp_cluster_wait();
  tc::tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
}

// ---------------------------------------------------------------------- plan
struct WeighPlan {
  bool tensor;
  int padded, ranges;
  size_t q_bytes, bytes;
};

WeighPlan wg_plan(const VbKv8WeighArgs *a) {
  WeighPlan pl = {};
  const long long rows = (long long)a->L * (a->q_heads / a->cache.kv_heads);
  const long long units = (long long)a->cache.batch * a->cache.kv_heads;
  pl.tensor = rows > 32;
  if (!pl.tensor) return pl;
  pl.padded = (int)((rows + WR_COLS - 1) / WR_COLS) * WR_COLS;
  // Key ranges per (sequence, head): the fewest waves of 74 pairs of CTAs, each with its
  // tiles and about two tiles' time for its start and end.
  const long long cap = (long long)a->cache.max_pages * a->cache.page;
  const long long tiles = ((cap < a->room ? cap : a->room) + WR_KEYS - 1) / WR_KEYS;
  double least = 1e300;
  pl.ranges = 1;
  for (int r = 1; r <= 74 && r <= tiles; ++r) {
    const double cost = (double)((units * r + 73) / 74) * (2 + (double)((tiles + r - 1) / r));
    if (cost < least) least = cost, pl.ranges = r;
  }
  pl.q_bytes = (size_t)units * pl.padded * a->cache.dim * 2;
  pl.bytes = pl.q_bytes + (size_t)units * pl.padded * sizeof(float2);
  return pl;
}

template <int D, int NR>
int wg_launch(const Kv8WeighParams &w, unsigned blocks, cudaStream_t s) {
  constexpr int SMEM = WG_WARPS * wg_stages<D>() * D * 16;
  static std::atomic<uint64_t> ready{0};
  const int rc = once_per_device(ready, [] {
    const cudaError_t e = cudaFuncSetAttribute(
        kv8_weigh_kernel<D, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    return e == cudaSuccess ? VB_OK
                            : set_error(VB_ERR_CUDA, "kv8_weigh_kernel attributes: %s",
                                        cudaGetErrorString(e));
  });
  if (rc != VB_OK) return rc;
  vb_launch(kv8_weigh_kernel<D, NR>, dim3(blocks, w.a.c.kv_heads, w.a.c.batch), dim3(WG_THREADS),
            SMEM, s, true, w);
  return check_launch("kv8_weigh_kernel");
}

template <int D>
int wg_run(Kv8WeighParams &w, const WeighPlan &pl, cudaStream_t s) {
  const VbKv8Cache &c = w.a.c;
  const long long cap = (long long)c.max_pages * c.page;
  const long long keys = cap < w.room ? cap : w.room, per = WG_WARPS * 16;
  const long long units = (long long)c.batch * c.kv_heads;
  if (keys == 0) return VB_OK;
  if (pl.tensor) {
    using S = WrShape<D>;
    static std::atomic<uint64_t> ready{0};
    const int rc = once_per_device(ready, [] {
      cudaFuncAttributes fa;
      cudaError_t e = cudaFuncGetAttributes(&fa, kv8_weigh_rows_kernel<D>);
      // the warpgroups' register shares are parts of what the block is launched with
      if (e == cudaSuccess && fa.numRegs != WR_REGS)
        return set_error(VB_ERR_CUDA, "kv8_weigh_rows_kernel: built with %d registers, %d needed",
                         fa.numRegs, WR_REGS);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(
          kv8_weigh_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
      return e == cudaSuccess ? VB_OK
                              : set_error(VB_ERR_CUDA, "kv8_weigh_rows_kernel attributes: %s",
                                          cudaGetErrorString(e));
    });
    if (rc != VB_OK) return rc;
    const long long rows = units * pl.padded, rpc = 256 * 8 / D;
    vb_launch(kv8_weigh_q_kernel<D>, dim3((unsigned)((rows + rpc - 1) / rpc)), dim3(256), 0, s, true,
              w);
    const int rc2 = check_launch("kv8_weigh_q_kernel");
    if (rc2 != VB_OK) return rc2;
    vb_launch(kv8_weigh_rows_kernel<D>, dim3((unsigned)(2 * units * w.ranges)), dim3(WR_THREADS),
              S::SMEM, s, true, w);
    return check_launch("kv8_weigh_rows_kernel");
  }
  // Groups of a warp: 8, fewer while that leaves SMs without work.
  w.groups = 8;
  while (w.groups > 1 && (keys + per * w.groups - 1) / (per * w.groups) * units < 148 * 4)
    w.groups /= 2;
  const unsigned blocks = (unsigned)((keys + per * w.groups - 1) / (per * w.groups));
  const int rows = w.a.L * w.a.rep;
  return rows <= 8 ? wg_launch<D, 1>(w, blocks, s)
         : rows <= 16 ? wg_launch<D, 2>(w, blocks, s)
                      : wg_launch<D, 4>(w, blocks, s);
}

int wg_check(const VbKv8WeighArgs *a) {
  VB_REQUIRE(a, "vb_kv8_weigh: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_weigh");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->q_heads >= 1 && a->q_heads % a->cache.kv_heads == 0 &&
                 a->q_heads / a->cache.kv_heads <= 128,
             "vb_kv8_weigh: %d query heads over %d kv heads (at most 128 each)", a->q_heads,
             a->cache.kv_heads);
  VB_REQUIRE(a->L >= 0 && (long long)a->L * a->q_heads <= 1 << 24,
             "vb_kv8_weigh: L=%d rows of %d heads", a->L, a->q_heads);
  VB_REQUIRE((long long)a->cache.batch * a->cache.kv_heads <= 1 << 21 &&
                 (long long)a->cache.batch * a->q_heads * a->L <= 1 << 28,
             "vb_kv8_weigh: %d sequences of %d kv heads, %d rows of %d heads each", a->cache.batch,
             a->cache.kv_heads, a->L, a->q_heads);
  VB_REQUIRE(a->room >= 0 && a->room <= 0x7fffffff - 65536, "vb_kv8_weigh: room=%d", a->room);
  // (a CTA counts its tiles of 256 rows by 256 keys in 31 bits)
  const long long cap = (long long)a->cache.max_pages * a->cache.page;
  const long long rows = (long long)a->L * (a->q_heads / a->cache.kv_heads);
  VB_REQUIRE((rows / 256 + 1) * ((cap < a->room ? cap : a->room) / 256 + 1) <= 0x7fffffff,
             "vb_kv8_weigh: %lld query rows of a kv head over %d keys", rows, a->room);
  return VB_OK;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

size_t vb_kv8_weigh_workspace_size(const VbKv8WeighArgs *a) {
  return wg_check(a) == VB_OK ? wg_plan(a).bytes : 0;
}

int vb_kv8_weigh(const VbKv8WeighArgs *a, vb_stream_t stream) {
  const int rc = wg_check(a);
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->lens && (a->L == 0 || (a->q && a->lse)) && (a->weights || a->room == 0),
             "vb_kv8_weigh: null tensor");
  VB_REQUIRE(!a->positions || a->seen, "vb_kv8_weigh: positions without seen");
  VB_REQUIRE(a->scale > 0.f && a->scale < 1e30f, "vb_kv8_weigh: scale %g", (double)a->scale);
  const WeighPlan pl = wg_plan(a);
  if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes))
    return set_error(VB_ERR_WORKSPACE, "vb_kv8_weigh: workspace %zu < %zu bytes",
                     a->workspace_bytes, pl.bytes);
  VB_REQUIRE(((uintptr_t)a->workspace % 16) == 0, "vb_kv8_weigh: workspace alignment");
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
  w.q16 = static_cast<uint16_t *>(a->workspace);
  w.row = reinterpret_cast<float2 *>(static_cast<uint8_t *>(a->workspace) + pl.q_bytes);
  w.padded = pl.padded; w.ranges = pl.ranges;
  cudaStream_t s = as_stream(stream);
  switch (a->cache.dim) {
    case 64: return wg_run<64>(w, pl, s);
    case 128: return wg_run<128>(w, pl, s);
    default: return wg_run<256>(w, pl, s);
  }
}

}  // extern "C"
