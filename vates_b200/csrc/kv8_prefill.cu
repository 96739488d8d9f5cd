// Attention over the paged 8-bit KV cache, many query rows per kv head
// (prompts and prompt chunks): 5th-generation tensor cores (tcgen05, float32
// accumulators in TMEM), tensor-core-bound.
//
//   z = scale * s_K(page) * (q . code_K),  o = sum_j 2^(z_j log2 e - m) s_V(page_j) code_V / l
//
// One CTA per SM owns NT row tiles of 128 query rows of one kv head (rows are
// the flattened (query, head of the group) pairs, so any group size fills them)
// and a range of keys in tiles of 128. The codes are exact in f16, and so are
// the queries after a power of two per row: both products are f16 with float32
// sums. Roles (four warpgroups):
//   * converters read the int8 rows from global memory (registers, one tile
//     ahead; page numbers two ahead) and write them as f16 operands in 128-byte
//     swizzled shared memory: K K-major, V as it lies (MN-major operand);
//   * one thread issues S = Q K^T of the next (key tile, row tile) item before
//     O += P V of the current one, so the tensor core works while the softmax
//     runs; the two S slots alternate;
//   * a softmax warpgroup per row tile (a thread per row = TMEM lane; for one
//     row tile two warpgroups would have to split the row) takes S, keeps a
//     running maximum that only moves when it grows by more than 2^4 (then O
//     and l are rescaled), and stores P = 2^(z - m) s_V / v over S in TMEM as
//     the f16 A operand of the second product. v is a power of two at least
//     every V scale so far. l is summed in float32 from the unrounded weights.
// A wait names the n-th completion of a barrier by its parity alone, so when it
// begins, completion n - 1 must have happened and n + 1 must not: S of an item
// waits for O of the last item in its slot, and the last O of a row tile has a
// barrier of its own.
// NT = 2 for head sizes 64 and 128, 1 for 256 (TMEM: 2 x 128 columns of S and
// NT * D of O are all 512). Every wait is bounded (2 s, then VB_STATUS_TIMEOUT).
#include "kv8_attn.cuh"
#include "tc100.cuh"

namespace vb {
namespace {

constexpr int KP_THREADS = 512;
constexpr int KP_KT = 128;              // keys per tile
constexpr int KP_BLOCK = 16384;         // 128 rows x 64 f16, 128-byte swizzle
constexpr uint64_t KP_WAIT_NS = 2000000000ull;
// Weights as f16 are 2^(z - m + shift) s_V / v, at most 2^15.5. A range of one
// tile knows its maximum and its largest V scale at once and uses all of that;
// a longer one leaves room for the maximum to grow by KP_MOVE (in log2) before
// O has to be rescaled. f16 keeps 11 bits down to 2^-14, so weights down to
// 2^-25 (2^-29) of the largest are as exact as the largest, and 2^-35 is the
// smallest that is kept.
constexpr float KP_SHIFT_ONE = 15.5f;
constexpr float KP_SHIFT = 11.f;
constexpr float KP_MOVE = 4.f;
constexpr float KP_NO_SCALE = -1000.f;  // log2 of the V scale of an all-zero page

template <int D>
struct KpShape {
  static constexpr int NT = D == 256 ? 1 : 2;       // row tiles
  static constexpr int STAGES = D == 256 ? 1 : 2;   // K, and V, operand tiles
  static constexpr int CONV_WG = D == 256 ? 2 : 1;  // converter warpgroups
  static constexpr int BLK = D / 64;                // 64-dim blocks of an operand tile
  static constexpr int TILE = BLK * KP_BLOCK;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = NT * TILE;
  static constexpr int V_OFF = K_OFF + STAGES * TILE;
  static constexpr int SMEM = V_OFF + STAGES * TILE + 1024;
  // registers per thread of the warpgroups; 128 at launch
  static constexpr int R_MMA = 40;
  static constexpr int R_CONV = D == 256 ? 120 : 104;
  static constexpr int R_SOFT = D == 256 ? 232 : 184;
  static_assert(R_MMA + CONV_WG * R_CONV + NT * R_SOFT == 4 * 128, "register shares");
};

// Byte offset of 16-byte chunk c of row r in a 128-row x 64-column block.
__device__ __forceinline__ uint32_t kp_sw(int r, int c) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}
// MN-major operand, 128-byte swizzle: lines of 64 elements along N, 8-line
// groups along K 1024 bytes apart, 64-element column blocks KP_BLOCK apart.
__device__ __forceinline__ uint64_t kp_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(KP_BLOCK >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__host__ __device__ constexpr uint32_t kp_idesc(int N, bool b_mn) {  // f16 x f16 -> f32, M = 128
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
// D[tmem] += A[tmem] * B[smem].
__device__ __forceinline__ void kp_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void kp_tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void kp_tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void kp_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void kp_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// The order of volatile statements is kept, so a group's exponentials are issued
// back to back.
__device__ __forceinline__ float kp_ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kp_max3(uint32_t a, uint32_t b, uint32_t c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;"
      : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return r;
}

struct KpBarriers {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2],
      o_last[2];
};

template <int D>
__global__ void __launch_bounds__(KP_THREADS, 1) kv8_prefill_kernel(Kv8AttnParams p) {
  using H = KpShape<D>;
  constexpr int NT = H::NT, ST = H::STAGES, ROWS = 128 * NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ __align__(8) KpBarriers bar;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float s_fac[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's rows and keys
  const int split = blockIdx.x % p.splits;
  const int rt = p.row_tiles - 1 - blockIdx.x / p.splits;  // longest (causal) rows first
  const int h = blockIdx.y, b = blockIdx.z;
  const int r_base = rt * ROWS, rows = p.L * p.rep;
  const Kv8Span sp = kv8_span(p, b, blockIdx.x == 0 && h == 0 && tid == 0);
  const int i_last = min(min(r_base + ROWS, rows) - 1, sp.q_len * p.rep - 1) / p.rep;
  const int kend = r_base < sp.q_len * p.rep ? sp.visible(i_last) : 0;
  const int tiles = (kend + KP_KT - 1) / KP_KT;
  const int share = tiles / p.splits, rest = tiles % p.splits;
  const int t0 = split * share + min(split, rest);
  const int t1 = t0 + share + (split < rest);
  const int n_items = (t1 - t0) * NT;
  const size_t tile_id = (((size_t)b * p.c.kv_heads + h) * p.row_tiles + rt) * p.splits + split;
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&bar.k_full[i], 4 * H::CONV_WG);
      tc::mbar_init(&bar.v_full[i], 4 * H::CONV_WG);
      tc::mbar_init(&bar.k_empty[i], 1);
      tc::mbar_init(&bar.v_empty[i], 1);
      tc::mbar_init(&bar.s_full[i], 1);
      tc::mbar_init(&bar.p_full[i], 4);
      tc::mbar_init(&bar.o_done[i], 1);
      tc::mbar_init(&bar.o_last[i], 1);
    }
    s_abort = 0;
    tc::fence_mbar_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(&s_tmem, 512);
    tc::tmem_relinquish();
  }

  // ---- queries: D / 8 lanes per row, f16 after the row's power of two; all
  // loads before the first use
  {
    constexpr int LPR = D / 8, PASS = KP_THREADS / LPR, NP = ROWS / PASS;
    const int c8 = tid % LPR;
    uint4 w[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int R = r_base + tid / LPR + k * PASS, i = p.row_of(R), hr = R - i * p.rep;
      w[k] = make_uint4(0, 0, 0, 0);
      if (n_items > 0 && R < rows && i < sp.q_len)
        w[k] = kv8_load8(p.q + b * p.qb + (int64_t)(h * p.rep + hr) * p.qh + (int64_t)i * p.ql +
                             c8 * 8,
                         p.vec);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int r = tid / LPR + k * PASS;
      const float pw = kv8_q_scale<LPR>(w[k]);
      if (c8 == 0) s_fac[r] = p.scale_log2 / pw;
      *reinterpret_cast<uint4 *>(smem + H::Q_OFF + (r >> 7) * H::TILE + (c8 >> 3) * KP_BLOCK +
                                 kp_sw(r & 127, c8 & 7)) = w[k];
    }
  }
  tc::fence_proxy_async_smem();
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int *abort = &s_abort;
  const uint32_t sbase = tc::smem_u32(smem);

  if (wg == 0) {
    // ================================================== tensor-core issuer
    kp_regs_dec<H::R_MMA>();
    if (tid == 0) {
      constexpr uint32_t ID_S = kp_idesc(KP_KT, false), ID_O = kp_idesc(D, true);
      auto wait = [&](uint64_t *m, int n) {  // n-th completion (from 0) of a barrier
        if (!tc::mbar_wait(m, (uint32_t)(n & 1), abort, KP_WAIT_NS)) {
          s_abort = 1;
          return false;
        }
        return true;
      };
      int s_sent = 0, o_sent = 0;
      bool ok = true;
      for (int w = 0; w <= n_items && ok; ++w) {
        if (w < n_items) {  // S of item w
          const int kt = w / NT, tile = w % NT, st = kt % ST;
          // the slot's P has been read: O of item w - 2 is done
          if (w >= 2) ok = wait(&bar.o_done[tile], (w - 2) / NT);
          if (tile == 0) ok = ok && wait(&bar.k_full[st], kt / ST);
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t qa = sbase + H::Q_OFF + tile * H::TILE;
          const uint32_t ka = sbase + H::K_OFF + st * H::TILE;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t o = (kk >> 2) * KP_BLOCK + (kk & 3) * 32;
            tc::mma_bf16_ss(tmem + (w & 1) * 128, tc::smem_desc_sw128(qa + o),
                            tc::smem_desc_sw128(ka + o), ID_S, kk > 0 ? 1u : 0u);
          }
          tc::mma_commit(&bar.s_full[w & 1]);
          if (tile == NT - 1) tc::mma_commit(&bar.k_empty[st]);
          ++s_sent;
        }
        if (w > 0) {  // O += P V of item w - 1
          const int v = w - 1, kt = v / NT, tile = v % NT, st = kt % ST;
          if (tile == 0) ok = wait(&bar.v_full[st], kt / ST);
          ok = ok && wait(&bar.p_full[v & 1], v >> 1);
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t va = sbase + H::V_OFF + st * H::TILE;
#pragma unroll
          for (int kk = 0; kk < KP_KT / 16; ++kk)
            kp_mma_ts(tmem + 256 + tile * D, tmem + (v & 1) * 128 + kk * 8,
                      kp_desc_mn(va + kk * 2048), ID_O, (kt > 0 || kk > 0) ? 1u : 0u);
          tc::mma_commit(&bar.o_done[tile]);
          if (v >= n_items - NT) tc::mma_commit(&bar.o_last[tile]);
          if (tile == NT - 1) tc::mma_commit(&bar.v_empty[st]);
          ++o_sent;
        }
      }
      // nothing of this CTA may be in flight when TMEM is freed
      for (int w = max(0, s_sent - 2); w < s_sent; ++w)
        if (!tc::mbar_wait(&bar.s_full[w & 1], (uint32_t)((w >> 1) & 1), nullptr, KP_WAIT_NS))
          s_abort = 1;
      for (int v = max(0, o_sent - NT); v < o_sent; ++v)
        if (!tc::mbar_wait(&bar.o_done[v % NT], (uint32_t)((v / NT) & 1), nullptr, KP_WAIT_NS))
          s_abort = 1;
    }
    __syncwarp();
  } else if (wg <= H::CONV_WG) {
    // ================================================== converters
    kp_regs_dec<H::R_CONV>();
    constexpr int CT = 128 * H::CONV_WG, CPR = D / 16, STEP = CT / CPR, NC = KP_KT / STEP;
    const int ctid = tid - 128;
    const int ch = ctid % CPR, key0 = ctid / CPR;
    uint4 kr[NC], vr[NC];
    // pool page of the 16-key group lane % 8 of tile t; rows without a page (past
    // the last key, or flagged) read page 0: their weights are 0
    auto group_page = [&](int t) {
      const int key = t * KP_KT + (lane & 7) * 16;
      return t < t1 && key < kend
                 ? max(0, kv8_page(table, p.c.max_pages, p.c.pages, key >> p.shift, p.status)) : 0;
    };
    const size_t pool_step = (size_t)p.c.kv_heads * p.c.page * D;
    const int8_t *kbase = p.c.k_codes + (size_t)h * p.c.page * D + ch * 16;
    const int8_t *vbase = p.c.v_codes + (size_t)h * p.c.page * D + ch * 16;
    auto load = [&](uint4 (&x)[NC], const int8_t *base, int id) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int key = key0 + i * STEP;  // a tile starts on a page boundary (page <= 128)
        const int pg = __shfl_sync(0xffffffffu, id, key >> 4);
        x[i] = ldg_nc_v4(base + pg * pool_step + (key & (p.c.page - 1)) * D);
      }
    };
    // 16 codes -> two 16-byte chunks; neighbouring 64-dim blocks store them in
    // opposite order so that the eight lanes of a store pass hit all banks
    auto store = [&](const uint4 (&x)[NC], uint8_t *tile) {
      const int e0 = (ch >> 2) & 1;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int key = key0 + i * STEP;
        uint4 o[2];
        const uint32_t w[4] = {x[i].x ^ 0x80808080u, x[i].y ^ 0x80808080u, x[i].z ^ 0x80808080u,
                               x[i].w ^ 0x80808080u};
        o[0] = make_uint4(h2_codes(__byte_perm(w[0], 0x64646464u, 0x4140)),
                          h2_codes(__byte_perm(w[0], 0x64646464u, 0x4342)),
                          h2_codes(__byte_perm(w[1], 0x64646464u, 0x4140)),
                          h2_codes(__byte_perm(w[1], 0x64646464u, 0x4342)));
        o[1] = make_uint4(h2_codes(__byte_perm(w[2], 0x64646464u, 0x4140)),
                          h2_codes(__byte_perm(w[2], 0x64646464u, 0x4342)),
                          h2_codes(__byte_perm(w[3], 0x64646464u, 0x4140)),
                          h2_codes(__byte_perm(w[3], 0x64646464u, 0x4342)));
        uint8_t *base = tile + (ch >> 2) * KP_BLOCK;
        const int c = 2 * (ch & 3);
        *reinterpret_cast<uint4 *>(base + kp_sw(key, c + e0)) = e0 ? o[1] : o[0];
        *reinterpret_cast<uint4 *>(base + kp_sw(key, c + 1 - e0)) = e0 ? o[0] : o[1];
      }
    };
    auto publish = [&](uint64_t *full) {
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(full);
    };
    // K runs a tile ahead of V: S of the next tile is issued before O of this one
    auto wait = [&](uint64_t *m, int n) {  // n-th completion of a barrier (n < 0: none needed)
      if (n >= 0 && !tc::mbar_wait(m, (uint32_t)(n & 1), abort, KP_WAIT_NS)) s_abort = 1;
      return !__any_sync(0xffffffffu, *abort != 0);
    };
    int id_v = group_page(t0), id_k = group_page(t0 + 1);  // of tiles n + 1 and n + 2
    load(kr, kbase, id_v);
    load(vr, vbase, id_v);
    bool ok = true;
    for (int n = -1; n < t1 - t0; ++n) {  // K of tile n + 1, V of tile n
      const int id_next = group_page(t0 + n + 3);
      if (n + 1 < t1 - t0) {
        const int st = (n + 1) % ST;
        ok = wait(&bar.k_empty[st], (n + 1) / ST - 1);
        if (!ok) break;
        store(kr, smem + H::K_OFF + st * H::TILE);
        publish(&bar.k_full[st]);
        load(kr, kbase, id_k);
      }
      if (n >= 0) {
        const int st = n % ST;
        ok = wait(&bar.v_empty[st], n / ST - 1);
        if (!ok) break;
        store(vr, smem + H::V_OFF + st * H::TILE);
        publish(&bar.v_full[st]);
        load(vr, vbase, id_v);
      }
      id_v = id_k;
      id_k = id_next;
    }
  } else {
    // ================================================== softmax, a thread per row
    kp_regs_inc<H::R_SOFT>();
    const int tile = wg - 1 - H::CONV_WG;
    const int r = tile * 128 + (tid & 127), R = r_base + r;
    const int vis = R < rows ? sp.visible(p.row_of(R)) : 0;
    const float fac = s_fac[r];
    const uint32_t trow = tmem + (((uint32_t)(warp & 3) * 32u) << 16);
    const bool one = t1 - t0 == 1;
    const float shift = one ? KP_SHIFT_ONE : KP_SHIFT;
    float m = -INFINITY, l = 0.f, lvref = KP_NO_SCALE;
    // scales of the 16-key group lane % 8 of a tile: K scale (-1: no such page)
    // and log2 of the V scale, loaded a tile ahead, page numbers two ahead
    auto group_page = [&](int t) {
      const int key = t * KP_KT + (lane & 7) * 16;
      return t < t1 && key < kend
                 ? kv8_page(table, p.c.max_pages, p.c.pages, key >> p.shift, nullptr) : -1;
    };
    auto group_scales = [&](int id, float &ks, float &vs) {
      ks = id >= 0 ? __ldg(p.c.k_scales + (size_t)id * p.c.kv_heads + h) : -1.f;
      vs = id >= 0 ? __ldg(p.c.v_scales + (size_t)id * p.c.kv_heads + h) : 0.f;
    };
    float ks_n, vs_n;
    group_scales(group_page(t0), ks_n, vs_n);
    int id_n = group_page(t0 + 1);
    bool ok = true;
    for (int t = t0; t < t1; ++t) {
      const int n = t - t0, w = n * NT + tile, slot = w & 1;
      const float ks_l = ks_n, lv_l = vs_n > 0.f ? log2f(vs_n) : KP_NO_SCALE;
      group_scales(id_n, ks_n, vs_n);
      id_n = group_page(t + 2);
      // v: a power of two at least every V scale so far
      float lv_top = lv_l;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1)
        lv_top = fmaxf(lv_top, __shfl_xor_sync(0xffffffffu, lv_top, o));
      const float lv_new = one ? lv_top : fmaxf(lvref, ceilf(lv_top));
      const uint32_t missing = __ballot_sync(0xffffffffu, ks_l < 0.f) & 0xFFu;

      if (!tc::mbar_wait(&bar.s_full[slot], (uint32_t)((w >> 1) & 1), abort, KP_WAIT_NS))
        s_abort = 1;
      ok = !__any_sync(0xffffffffu, *abort != 0);
      if (!ok) break;
      tc::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tc::tmem_ld32(trow + slot * 128 + q * 32, s[q]);
      tc::tmem_ld_wait();
      const int lim = vis - t * KP_KT;  // visible keys of this tile
      if (lim < KP_KT || missing) {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const bool gone = (missing >> g) & 1;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (gone || g * 16 + j >= lim) s[g >> 1][(g & 1) * 16 + j] = 0xFF800000u;
        }
      }
      float f[8];
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const float ks = __shfl_sync(0xffffffffu, ks_l, g);
        // scale 0: every code of the page is 0 (1 keeps -inf * 0 out)
        f[g] = fac * (ks > 0.f ? ks : 1.f);
        const uint32_t *v = s[g >> 1] + (g & 1) * 16;
        float x0 = kp_max3(v[0], v[1], v[2]), x1 = kp_max3(v[3], v[4], v[5]);
        float x2 = kp_max3(v[6], v[7], v[8]), x3 = kp_max3(v[9], v[10], v[11]);
        x0 = kp_max3(__float_as_uint(x0), v[12], v[13]);
        x1 = kp_max3(__float_as_uint(x1), v[14], v[15]);
        top = fmaxf(top, fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * f[g]);
      }
      const bool move = top > m + KP_MOVE;
      const float to = move ? top : m;
      const float alpha = move ? kv8_ex2(m - to) : 1.f;
      m = to;
      l *= alpha;
      if (n > 0 && (lv_new > lvref || __any_sync(0xffffffffu, move))) {  // rescale O
        if (!tc::mbar_wait(&bar.o_done[tile], (uint32_t)((n - 1) & 1), abort, KP_WAIT_NS))
          s_abort = 1;
        ok = !__any_sync(0xffffffffu, *abort != 0);
        if (!ok) break;
        tc::tc_fence_after();
        const float a = alpha * kv8_ex2(lvref - lv_new);
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t v[32];
          tc::tmem_ld32(trow + 256 + tile * D + c0, v);
          tc::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
          kp_tmem_st32(trow + 256 + tile * D + c0, v);
        }
        kp_tmem_st_wait();
      }
      lvref = lv_new;
      const float sub = shift - (m == -INFINITY ? 0.f : m);
      // Groups of 16: the arguments of the next one are formed before this one's
      // exponentials are used, so that a warp alone on its scheduler does not
      // wait for each.
      float x[2][16], cg[8];
      auto arguments = [&](int g) {
        const float lv = __shfl_sync(0xffffffffu, lv_l, g);
        cg[g] = lv > KP_NO_SCALE ? lv - lvref : 0.f;
        const f2 ff = f2_make(f[g], f[g]), cc = f2_make(sub + cg[g], sub + cg[g]);
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const uint32_t *v = s[g >> 1] + (g & 1) * 16 + j;
          f2_split(f2_fma(f2_make(__uint_as_float(v[0]), __uint_as_float(v[1])), ff, cc),
                   x[g & 1][j], x[g & 1][j + 1]);
        }
      };
      arguments(0);
      uint32_t pk[2][32];
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        float e[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) e[j] = kp_ex2(x[g & 1][j]);
        if (g < 7) arguments(g + 1);
        f2 sum0 = f2_make(e[0], e[1]), sum1 = f2_make(e[2], e[3]);
#pragma unroll
        for (int j = 4; j < 16; j += 4) {
          sum0 = f2_add(sum0, f2_make(e[j], e[j + 1]));
          sum1 = f2_add(sum1, f2_make(e[j + 2], e[j + 3]));
        }
        float s0, s1;
        f2_split(f2_add(sum0, sum1), s0, s1);
#pragma unroll
        for (int j = 0; j < 16; j += 2) pk[g >> 2][(g & 3) * 8 + (j >> 1)] = pack_h2(e[j], e[j + 1]);
        l = fmaf(s0 + s1, kp_ex2(fminf(-cg[g], 126.f)), l);
        if (g == 3) kp_tmem_st32(trow + slot * 128, pk[0]);
      }
      kp_tmem_st32(trow + slot * 128 + 32, pk[1]);
      kp_tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.p_full[slot]);
    }
    // ---- O of this tile's last product
    if (ok && t1 > t0) {
      if (!tc::mbar_wait(&bar.o_last[tile], 0, abort, KP_WAIT_NS)) s_abort = 1;
      ok = !__any_sync(0xffffffffu, *abort != 0);
      tc::tc_fence_after();
    }
    if (ok) {
      const float v = kv8_ex2(lvref);
      const int i = p.row_of(R), hr = R - i * p.rep;
      const size_t row = ((size_t)b * p.Hq + h * p.rep + hr) * p.L + i;
      const bool live = R < rows;
      if (p.splits > 1) {
        if (live) p.ml_part[tile_id * ROWS + r] = make_float2(m - shift, l);
      } else if (live && p.lse) {
        p.lse[row] = l == 0.f ? -INFINITY : (m - shift + log2f(l)) * 0.69314718055994531f;
      }
      const float inv = p.splits > 1 ? v : l == 0.f ? 0.f : v / l;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t x[32];
        if (t1 > t0) {
          tc::tmem_ld32(trow + 256 + tile * D + c0, x);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = 0;
        }
        float y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(x[j]) * inv;
        __syncwarp();
        if (!live) {
        } else if (p.splits > 1) {
          if (t1 > t0) {
            float4 *d4 = reinterpret_cast<float4 *>(p.o_part + (tile_id * ROWS + r) * D + c0);
#pragma unroll
            for (int q = 0; q < 8; ++q)
              d4[q] = make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
          }
        } else {
          uint4 *d4 = reinterpret_cast<uint4 *>(p.out + row * D + c0);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            d4[q] = make_uint4(pack_bf2(y[8 * q], y[8 * q + 1]), pack_bf2(y[8 * q + 2], y[8 * q + 3]),
                               pack_bf2(y[8 * q + 4], y[8 * q + 5]),
                               pack_bf2(y[8 * q + 6], y[8 * q + 7]));
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (tid == 0 && *abort) flag_status(p.status, VB_STATUS_TIMEOUT);
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

template <int D>
int kp_launch(const Kv8AttnParams &p, cudaStream_t s) {
  using H = KpShape<D>;
  static bool ready = false;
  if (!ready) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kv8_prefill_kernel<D>);
    // the warpgroups' register shares add up to 128 per thread at launch
    if (e == cudaSuccess && fa.numRegs != 128)
      return set_error(VB_ERR_CUDA, "kv8_prefill_kernel: built with %d registers, 128 needed",
                       fa.numRegs);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kv8_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               H::SMEM);
    if (e != cudaSuccess)
      return set_error(VB_ERR_CUDA, "kv8_prefill_kernel attributes: %s", cudaGetErrorString(e));
    ready = true;
  }
  vb_launch(kv8_prefill_kernel<D>, dim3(p.row_tiles * p.splits, p.c.kv_heads, p.c.batch),
            dim3(KP_THREADS), H::SMEM, s, true, p);
  return check_launch("kv8_prefill_kernel");
}

}  // namespace

int kv8_prefill_rows(int dim) { return dim == 256 ? KpShape<256>::NT * 128 : 256; }

int kv8_prefill_launch(const Kv8AttnParams &p, cudaStream_t s) {
  switch (p.c.dim) {
    case 64: return kp_launch<64>(p, s);
    case 128: return kp_launch<128>(p, s);
    default: return kp_launch<256>(p, s);
  }
}

}  // namespace vb
