// Attention over the paged 8-bit KV cache, many query rows per kv head
// (prompts and prompt chunks): 5th-generation tensor cores (tcgen05, float32
// accumulators in TMEM), tensor-core-bound.
//
//   z = scale * s_K(page) * (q . code_K),  o = sum_j 2^(z_j log2 e - m) s_V(page_j) code_V / l
//
// A pair of CTAs on two SMs (a cluster; tcgen05 cta_group::2) owns 256 query rows
// of one kv head, 128 each (rows are the flattened (query, head of the group)
// pairs, so any group size fills them), and a range of keys in tiles of 128.
// Each CTA converts and holds half of every K tile (64 keys) and half of every V
// tile (half of the dims) for both: half the loads, conversions and shared-memory
// reads that a CTA on its own would need (4,096 rows over 32,768 keys of 256:
// 2.4 ms). The codes are exact in f16, and so are the queries after a power of
// two per row: both products are f16 with float32 sums. Roles (warpgroups):
//   * converters read the int8 rows from global memory into registers (K a tile
//     ahead of V, page numbers another tile ahead) and write them as f16 operands
//     in 128-byte swizzled shared memory, two stages: K K-major, V as it lies
//     (MN-major operand);
//   * one thread of the pair issues S = Q K^T one key tile ahead of O += P V (two
//     for heads of 64 and 128, which leave TMEM columns for a third S slot), so the
//     tensor cores work while the softmax runs;
//   * two softmax warpgroups per CTA, a thread per row, take the key tiles in
//     turn: one's exponentials run while the other waits for its products. What a
//     tile needs of the one before it is the running maximum, which is handed
//     over before the exponentials. It only moves when it grows by more than 2^9
//     (then O is rescaled), and P = 2^(z - m) s_V / v goes over S in TMEM as the
//     f16 A operand of the second product (the codes are f16, so the weights have to
//     be; an eighth of what out loses to bf16). v is a power of two at least every V
//     scale so far. l is summed in float32 from the unrounded weights.
// A wait names the n-th completion of a barrier by its parity alone, so when it
// begins, completion n - 1 must have happened and n + 1 must not: S of a tile
// waits for O of the last tile in its slot, and the last O and the end have
// barriers of their own. Every wait is bounded (2 s, then VB_STATUS_TIMEOUT).
//
// What bounds it: 4,096 rows over 32,768 keys of 256 take 1.97 to 2.05 ms, 1.0
// PFLOP/s of the 1.7 that a library product reaches in a burst. A tile of 128 keys
// takes some 2.3 us, of which the products fill 1.45; the rest is the chain S, maximum,
// exponentials, O of one tile, of which only two are in TMEM (O takes the other half).
// For heads of 64 it is the softmax (a tile 1.1 us; exponentials alone fill 0.55). A
// launch without keys takes 4.6 us, one with a single tile 8.9 (heads of 256: 6.2, 13.6).
#include "kv8_attn.cuh"
#include "kv8_pair.cuh"

namespace vb {
namespace {

constexpr int KP_THREADS = 512;
constexpr int KP_KT = 128;              // keys per tile
constexpr int KP_STAGES = 2;            // K, and V, operand tiles
constexpr int KP_ROWS = 256;            // query rows of a pair of CTAs
// Weights as f16 are 2^(z - m) s_V / v, m the row's maximum less a shift, at most
// 2^15.5: m is rounded up and what a score may reach down, so that this holds for scores
// of any size. A range of one tile knows its maximum and its largest V scale at once and
// uses all of that; a longer one leaves room for the maximum to grow by KP_MOVE (in
// log2) before O has to be rescaled, which stalls the pair of CTAs (a shift of 11 and a
// move of 4 cost 6 % more time over 32,768 keys, a third more over 2,048). f16 keeps 11
// bits down to 2^-14, so weights down to 2^-20 (2^-29) of the largest are as exact as
// the largest, and 2^-30 is the smallest that is kept.
constexpr float KP_SHIFT_ONE = 15.5f;
constexpr float KP_SHIFT = 6.f;
constexpr float KP_MOVE = 9.f;
constexpr float KP_NO_SCALE = -1000.f;  // log2 of a V scale of 0

template <int D>
struct KpShape {
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int K_BLOCK = KP_BLOCK / 2;      // 64 keys x 64 dims
  static constexpr int K_HALF = 64 * D * 2;
  // Dims of this CTA's V half. Halves of 64 dims at least: for D = 64, CTA 0 holds
  // all of V and the columns of O from 64 on are not used.
  static constexpr int VD = D == 256 ? 128 : 64;
  static constexpr int V_HALF = 128 * VD * 2;
  // S slots in TMEM, 128 columns each, before the columns of O
  static constexpr int SLOTS = D == 256 ? 2 : 3, O_COL = SLOTS * 128;
  static constexpr int K_OFF = Q_BYTES;
  static constexpr int V_OFF = K_OFF + KP_STAGES * K_HALF;
  static constexpr int SMEM = V_OFF + KP_STAGES * V_HALF + 1024;
};
// Registers per thread of the four warpgroups; 128 at launch.
constexpr int KP_R_MMA = 56, KP_R_CONV = 136, KP_R_SOFT = 160;
static_assert(KP_R_MMA + KP_R_CONV + 2 * KP_R_SOFT == 4 * 128, "register shares");

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
// The order of volatile statements is kept, so a group's exponentials are issued
// back to back.
__device__ __forceinline__ float kp_ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kp_max3(uint32_t a, uint32_t b, uint32_t c) {
  float r;
  asm volatile("max.f32 %0, %1, %2, %3;"
      : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return r;
}

__device__ __forceinline__ void kp_mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem,
                                          uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
// The 256 softmax threads of a CTA meet; one half of them hands over to the other
// (`from`: the warpgroup that arrives).
__device__ __forceinline__ void kp_soft_sync() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
__device__ __forceinline__ void kp_hand_over(int from) {
  asm volatile("bar.arrive %0, 256;" ::"r"(1 + from) : "memory");
}
__device__ __forceinline__ void kp_take_over(int from) {
  asm volatile("bar.sync %0, 256;" ::"r"(1 + from) : "memory");
}
// 2^(a - b), 1 where both are the same (infinities too).
__device__ __forceinline__ float kp_ratio(float a, float b) { return a == b ? 1.f : kp_ex2(a - b); }
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
__device__ __forceinline__ void kp_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void kp_tmem_zero8(uint32_t taddr) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%1,%1,%1,%1,%1,%1,%1};" ::"r"(
                   taddr),
               "r"(0)
               : "memory");
}
__device__ __forceinline__ void kp_store32(float *p, const float *x) {  // one whole sector
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]),
               "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
__device__ __forceinline__ void kp_tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
struct KpBarriers {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[3], p_full[3], o_done[3], q_full, o_last, drain;
};

// Segments (kv8_attn.cuh): what a pair of CTAs is to do, from the rows that there are.
// Lengths are on the device, so the tiles and key ranges are dealt here: 64 sequences
// with 167 of 64 x 4 rows behind 32,768 keys, 16/2 heads of 256, fill 12 tiles instead of 16:
// 152 us for 211. It takes 2 us.
struct KpDeal {
  int4 seg;
  int tile, in_seg;    // row tile, of all and within the segment
  int h, split, splits;
};
// What is the same in all lanes, for the compiler to know: without it the roles' loops count
// as divergent, and a key tile takes half as long again.
__device__ __forceinline__ int kp_uniform(int x) {
  return (int)__reduce_max_sync(0xffffffffu, (unsigned)x);
}
// Key ranges per row tile for `base` row tiles of up to `tiles` key tiles, by the rule
// of kv8_ranges; the same in every lane.
__device__ __forceinline__ int kp_ranges(int base, int tiles, int pairs) {
  const int most = min(pairs, 8 * 74);
  if (base > most) return 1;
  // (32 x the time, of at most 8 waves; ranges of more than 2^16 tiles count as that long)
  auto cost = [&](int s) {
    return 32u * (unsigned)((base * s + 73) / 74) * (3 + min((tiles + s - 1) / s, 1 << 16)) +
           (s > 1 ? 64 + base * s : 0);
  };
  unsigned best = ~0u;
  int at = 1;
  for (int s = (threadIdx.x & 31) + 1; s <= min(74, tiles) && base * s <= most; s += 32)
    if (s > 1 && cost(s) < best) best = cost(s), at = s;
  const unsigned least = __reduce_min_sync(0xffffffffu, best);
  at = (int)__reduce_min_sync(0xffffffffu, best == least ? (unsigned)at : 74u);
  return least < cost(1) / 10 * 9 ? at : 1;
}
// False if there is nothing for the pair; the same for all threads of both CTAs. s_seg,
// s_tiles: KP_THREADS of them.
__device__ __forceinline__ bool kp_deal(const Kv8AttnParams &p, int4 *s_seg, int *s_tiles, KpDeal &d) {
  const int tid = threadIdx.x, lane = tid & 31, pair = blockIdx.x >> 1;
  const int lanes = p.seg_lanes, per = KP_THREADS / lanes;
  // row tiles of the segments from c0 on
  auto count = [&](int c0) {
    const int g = c0 + tid / lanes;
    int n = 0;
    if (g < p.n_segs) {
      const int4 s = p.segs[g];
      if ((tid & (lanes - 1)) == 0) s_seg[tid / lanes] = s;
      for (int m = tid & (lanes - 1); m < s.y; m += lanes)
        n += blockIdx.x == 0 ? kv8_span(p, s.x + m, true).q_len
                             : kv8_rows(p.q_lens, s.x + m, p.L, nullptr);
    }
    __syncwarp();
    for (int o = lanes / 2; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if ((tid & (lanes - 1)) == 0) s_tiles[tid / lanes] = (n * p.rep + KP_ROWS - 1) / KP_ROWS;
    __syncthreads();
  };
  const int H = p.c.kv_heads;
  if (!p.deal) {  // a row tile for each segment
    d.splits = p.splits;
    d.split = pair % d.splits;
    d.h = pair / d.splits % H;
    d.tile = pair / d.splits / H;
    d.in_seg = 0;
    d.seg = p.segs[d.tile];
    if (pair == 0 && tid == 0 && (blockIdx.x & 1) == 0) p.places[0] = d.splits;
    return true;
  }
  int total = 0;
  for (int c0 = 0; c0 < p.n_segs; c0 += per) {
    if (c0 > 0) __syncthreads();  // (the last ones have been read)
    count(c0);
    int n = 0;
    for (int i = lane; i < per; i += 32) n += s_tiles[i];
    total += __reduce_add_sync(0xffffffffu, n);
  }
  d.splits = kp_ranges(total * H, p.longest, p.pairs);
  if (pair == 0 && tid == 0 && (blockIdx.x & 1) == 0) p.places[0] = d.splits;
  if (pair >= (long long)total * H * d.splits) return false;
  d.split = pair % d.splits;
  d.h = pair / d.splits % H;
  d.tile = pair / d.splits / H;
  int before = 0;
  for (int c0 = 0; c0 < p.n_segs; c0 += per) {
    if (p.n_segs > per) {
      __syncthreads();
      count(c0);
    }
    for (int i = 0; i < per; i += 32) {  // (zeros behind the last segment)
      const int n = i + lane < per ? s_tiles[i + lane] : 0;
      int end = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, d.tile < before + end);
      if (past) {
        const int l = __ffs(past) - 1;
        d.seg = s_seg[i + l];
        d.in_seg = d.tile - before - __shfl_sync(0xffffffffu, end - n, l);
        return true;
      }
      before += __shfl_sync(0xffffffffu, end, 31);
    }
  }
  return false;  // (not reached)
}

// SEG: segments in the place of sequences.
template <int D, bool SEG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(KP_THREADS, 1)
    kv8_prefill_kernel(Kv8AttnParams p) {
  using H = KpShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~uintptr_t(1023));
  __shared__ __align__(8) KpBarriers bar;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float s_fac[128], s_m[128], s_l[2][128], s_lv[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
  if (!SEG) pdl_launch_dependents();
  pdl_wait();
  if (SEG) pdl_launch_dependents();  // (it may need what this one waited for)

  // ---- the pair's rows and keys, this CTA's rows r_base .. + 127
  const int rank = blockIdx.x & 1;
  int rt, split, h, b, rows, splits = p.splits;
  KpDeal deal = {};
  // What this CTA's rows are: sequence, query, head of the group, keys seen. (Where keys
  // come, after everyone has looked.)
  int4 *s_row = reinterpret_cast<int4 *>(smem + H::K_OFF);
  if constexpr (SEG) {
    // (in the operands' place)
    if (!kp_deal(p, reinterpret_cast<int4 *>(smem), reinterpret_cast<int *>(smem + 16 * KP_THREADS),
                 deal))
      return;
    rt = kp_uniform(deal.in_seg); split = kp_uniform(deal.split); splits = kp_uniform(deal.splits);
    h = kp_uniform(deal.h); b = 0;
    deal.tile = kp_uniform(deal.tile);
    deal.seg = make_int4(kp_uniform(deal.seg.x), kp_uniform(deal.seg.y), kp_uniform(deal.seg.z),
                         kp_uniform(deal.seg.w));
  } else {
    const int units = p.c.batch * p.c.kv_heads * splits, unit = (blockIdx.x >> 1) % units;
    rt = p.row_tiles - 1 - (blockIdx.x >> 1) / units;  // longest (causal) rows first
    split = unit % splits; h = unit / splits % p.c.kv_heads; b = unit / splits / p.c.kv_heads;
    rows = p.L * p.rep;
  }
  const int4 seg = deal.seg;
  const int pair_base = rt * KP_ROWS, r_base = pair_base + rank * 128;
  Kv8Span sp;
  int kend, owner = b;
  if constexpr (SEG) {
    // The tile's sequences, keys that its rows see, and a sequence that sees as many: its
    // table has them. Every warp looks at all sequences up to them, 32 at a time.
    int2 *s_seq = reinterpret_cast<int2 *>(s_row + 128);  // their first rows, sequences
    int n_seq = 0;
    kend = rows = 0;
    owner = seg.x;
    const bool flag = !p.deal && split == 0 && h == 0 && rank == 0 && warp == 0;
    for (int m = 0; m < seg.y && (!p.deal || rows < pair_base + KP_ROWS); m += 32) {
      const bool there = m + lane < seg.y;
      const int bq = seg.x + m + lane;
      int n = 0;
      if (there)
        n = flag ? kv8_span(p, bq, true).q_len : kv8_rows(p.q_lens, bq, p.L, nullptr);
      n *= p.rep;
      int end = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += up;
      }
      const int begin = rows + end - n;
      rows += __shfl_sync(0xffffffffu, end, 31);
      int seen = 0;
      if (n > 0 && begin < pair_base + KP_ROWS && begin + n > pair_base) {
        const Kv8Span s = kv8_span(p, bq, false);
        // (a row tile that ends or begins within a sequence may see less)
        seen = kv8_reach(seg, s.visible(s.q_len - 1));
        if (begin >= pair_base && split == 0 && h == 0 && rank == 0 && warp == 0)
          p.places[1 + bq] = deal.tile * KP_ROWS + begin - pair_base;
      }
      const int most = (int)__reduce_max_sync(0xffffffffu, (unsigned)seen);
      if (most > kend) {
        kend = most;
        owner = seg.x + m + __ffs(__ballot_sync(0xffffffffu, seen == most)) - 1;
      }
      const bool here = n > 0 && begin < r_base + 128 && begin + n > r_base;
      const uint32_t all = __ballot_sync(0xffffffffu, here);
      if (here && warp == 0) s_seq[n_seq + __popc(all & ((1u << lane) - 1))] = make_int2(begin, bq);
      n_seq += __popc(all);
    }
    rows = kp_uniform(rows);
    kend = kp_uniform(kend);
    owner = kp_uniform(owner);
    __syncthreads();
    if (tid < 128) {
      const int R = r_base + tid;
      int4 x = make_int4(seg.x, 0, 0, 0);
      if (R < rows) {
        int at = 0;  // the last sequence that begins at R or before
#pragma unroll
        for (int o = 64; o > 0; o >>= 1)
          if (at + o < n_seq && s_seq[at + o].x <= R) at += o;
        const int2 q = s_seq[at];
        x.x = q.y;
        x.y = p.row_of(R - q.x);
        x.z = R - q.x - x.y * p.rep;
        x.w = kv8_reach(seg, kv8_span(p, q.y, false).visible(x.y));
      }
      s_row[tid] = x;
    }
    __syncthreads();
  } else {
    sp = kv8_span(p, b, rt == p.row_tiles - 1 && split == 0 && rank == 0 && h == 0 && tid == 0);
    const int i_last = p.row_of(max(0, min(min(pair_base + KP_ROWS, rows), sp.q_len * p.rep) - 1));
    kend = pair_base < sp.q_len * p.rep ? sp.visible(i_last) : 0;
  }
  // The row R of the tile: sequence, query, head of the group, keys seen.
  auto row_at = [&](int R) {
    Kv8SegRow x;
    if constexpr (SEG) {
      const int4 v = s_row[R - r_base];
      x.b = v.x; x.i = v.y; x.hr = v.z; x.vis = v.w;
    } else {
      x.b = b;
      x.i = p.row_of(R);
      x.hr = R - x.i * p.rep;
      x.vis = R < rows && x.i < sp.q_len;  // (whether it is there; for queries only)
    }
    return x;
  };
  const int tiles = (kend + KP_KT - 1) / KP_KT;
  const int share = tiles / splits, rest = tiles % splits;
  const int t0 = split * share + min(split, rest);
  const int t1 = t0 + share + (split < rest);
  const int n_tiles = t1 - t0;
  const size_t tile_id =
      SEG ? blockIdx.x >> 1 : (((size_t)b * p.c.kv_heads + h) * p.row_tiles + rt) * splits + split;
  // (a segment's first key is the first of a page)
  const int pages_before = SEG ? seg.z >> p.shift : 0, table_len = p.c.max_pages - pages_before;
  const int32_t *table = p.c.page_table + (size_t)owner * p.c.max_pages + pages_before;

  if (tid == 32) {
    for (int i = 0; i < KP_STAGES; ++i) {
      tc::mbar_init(&bar.k_full[i], 2 * 4);   // converter warps of both CTAs
      tc::mbar_init(&bar.v_full[i], 2 * 4);
      tc::mbar_init(&bar.k_empty[i], 1);
      tc::mbar_init(&bar.v_empty[i], 1);
    }
    for (int i = 0; i < H::SLOTS; ++i) {
      tc::mbar_init(&bar.s_full[i], 1);
      tc::mbar_init(&bar.p_full[i], 2 * 4);   // softmax warps of a tile, both CTAs
      tc::mbar_init(&bar.o_done[i], 1);
    }
    tc::mbar_init(&bar.q_full, 2);  // both CTAs
    tc::mbar_init(&bar.o_last, 1);
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
  // Every role: barriers and TMEM of both CTAs are there. First loads come before it.
  uint32_t tmem = 0;
  auto ready = [&]() {
    tc::tc_fence_before();
    __syncthreads();
    kp_cluster_wait();
    tc::tc_fence_after();
    tmem = s_tmem;
  };
  volatile int *abort = &s_abort;
  const uint32_t sbase = tc::smem_u32(smem);
  // The warp waits for the n-th completion (from 0) of a barrier; false after a
  // wait of this CTA has given up.
  auto wait = [&](uint64_t *m, int n) {
    const bool there = tc::mbar_wait(m, (uint32_t)(n & 1), abort, KP_WAIT_NS);
    if (!there) s_abort = 1;
    return __all_sync(0xffffffffu, there);
  };

  if (wg == 0) {
    // ================================================== tensor-core issuer
    kp_regs_dec<KP_R_MMA>();
    ready();
    if (warp == 0 && rank == 0) {
      constexpr uint32_t ID_S = kp_idesc(KP_KT, false), ID_O = kp_idesc(2 * H::VD, true);
      const uint32_t one = kp_elect();
      // descriptors of the first 16-element step; a step adds to the address field
      const uint64_t q_desc = tc::smem_desc_sw128(sbase);
      const uint64_t k_desc = tc::smem_desc_sw128(sbase + H::K_OFF);
      const uint64_t v_desc = kp_desc_mn(sbase + H::V_OFF);
      bool ok = n_tiles == 0 || wait(&bar.q_full, 0);
      for (int w = 0; w < n_tiles + H::SLOTS - 1 && ok; ++w) {
        if (w < n_tiles) {  // S of tile w
          const int st = w % KP_STAGES, slot = w % H::SLOTS;
          // the slot's P has been read: O of tile w - SLOTS is done
          if (w >= H::SLOTS) ok = wait(&bar.o_done[slot], w / H::SLOTS - 1);
          ok = ok && wait(&bar.k_full[st], w / KP_STAGES);
          if (!ok) break;
          tc::tc_fence_after();
          const uint64_t kd = k_desc + st * (H::K_HALF >> 4);
          const uint32_t d = tmem + slot * 128;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            kp_mma_ss(one, d, q_desc + (((kk >> 2) * KP_BLOCK + (kk & 3) * 32) >> 4),
                      kd + (((kk >> 2) * H::K_BLOCK + (kk & 3) * 32) >> 4), ID_S,
                      kk > 0 ? 1u : 0u);
          kp_commit(one, &bar.s_full[slot]);
          kp_commit(one, &bar.k_empty[st]);
        }
        const int v = w - (H::SLOTS - 1);
        if (v >= 0) {  // O += P V of tile v
          const int st = v % KP_STAGES, slot = v % H::SLOTS;
          ok = wait(&bar.v_full[st], v / KP_STAGES) && wait(&bar.p_full[slot], v / H::SLOTS);
          if (!ok) break;
          tc::tc_fence_after();
          const uint64_t vd = v_desc + st * (H::V_HALF >> 4);
          const uint32_t a = tmem + slot * 128;
#pragma unroll
          for (int kk = 0; kk < KP_KT / 16; ++kk)
            kp_mma_ts(one, tmem + H::O_COL, a + kk * 8, vd + (kk * 2048 >> 4), ID_O,
                      kk > 0 ? 1u : (v > 0 ? 1u : 0u));
          kp_commit(one, &bar.o_done[slot]);
          if (v == n_tiles - 1) kp_commit(one, &bar.o_last);
          kp_commit(one, &bar.v_empty[st]);
        }
      }
      // nothing of the pair may be in flight when TMEM is freed
      kp_commit(one, &bar.drain);
      if (!tc::mbar_wait(&bar.drain, 0, nullptr, KP_WAIT_NS)) s_abort = 1;
    }
    __syncwarp();
  } else if (wg == 1) {
    // ================================================== converters
    kp_regs_inc<KP_R_CONV>();
    const int ctid = tid - 128;
    // K: 64 keys of all dims; V: 128 keys of half of the dims; 16 codes at a time
    constexpr int KC = D / 16, KSTEP = 128 / KC, KN = 64 / KSTEP;
    constexpr int VC = H::VD / 16, VSTEP = 128 / VC, VN = 128 / VSTEP;
    const int kch = ctid % KC, kkey = ctid / KC, vch = ctid % VC, vkey = ctid / VC;
    uint4 kr[KN], vr[VN];
    // table entry of the 16-key group lane % 8 of tile t, and later its pool page;
    // rows without one (past the last key, or flagged) read page 0: their weights
    // are 0
    auto group_entry = [&](int t) {
      const int key = t * KP_KT + (lane & 7) * 16;
      return t < t1 && key < kend ? kv8_page_load(table, table_len, key >> p.shift) : 0;
    };
    // (segments: the head's page, counted over all heads: h, which was dealt, costs registers
    // in the bases, for heads of 256 31 of the rows on their way and a key tile a sixth)
    auto group_page = [&](int entry) {
      const int id = max(0, kv8_page_ok(entry, p.c.pages, p.status));
      return SEG ? id * p.c.kv_heads + h : id;
    };
    const size_t pool_step = (size_t)(SEG ? 1 : p.c.kv_heads) * p.c.page * D;
    const size_t head = SEG ? 0 : (size_t)h * p.c.page * D;
    const int8_t *kbase = p.c.k_codes + head + kch * 16;
    const int8_t *vbase = p.c.v_codes + head + rank * H::VD + vch * 16;
    auto load_k = [&](int id) {
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        const int key = rank * 64 + kkey + i * KSTEP;  // a tile starts on a page boundary
        const int pg = __shfl_sync(0xffffffffu, id, key >> 4);
        kr[i] = ldg_nc_v4(kbase + pg * pool_step + (key & (p.c.page - 1)) * D);
      }
    };
    auto load_v = [&](int id) {
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const int key = vkey + i * VSTEP;
        const int pg = __shfl_sync(0xffffffffu, id, key >> 4);
        vr[i] = ldg_nc_v4(vbase + pg * pool_step + (key & (p.c.page - 1)) * D);
      }
    };
    auto publish = [&](uint64_t *full) {
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) kp_arrive_leader(full);
    };
    const bool has_v = D > 64 || rank == 0;
    // of tiles n + 1 and n + 2
    int id_v = group_page(group_entry(t0)), id_k = group_page(group_entry(t0 + 1));
    load_k(id_v);
    if (has_v) load_v(id_v);
    ready();
    for (int n = -1; n < n_tiles; ++n) {  // K of tile n + 1, V of tile n
      const int entry = group_entry(t0 + n + 3);
      if (n + 1 < n_tiles) {
        const int st = (n + 1) % KP_STAGES;
        if (n + 1 >= KP_STAGES && !wait(&bar.k_empty[st], (n + 1) / KP_STAGES - 1)) break;
        uint8_t *tile = smem + H::K_OFF + st * H::K_HALF;
#pragma unroll
        for (int i = 0; i < KN; ++i) kp_store_codes(kr[i], tile, H::K_BLOCK, kkey + i * KSTEP, kch);
        publish(&bar.k_full[st]);
      }
      const int id_next = group_page(entry);  // before rows are asked for: it would wait for them
      if (n + 1 < n_tiles) load_k(id_k);
      if (n >= 0) {
        const int st = n % KP_STAGES;
        if (n >= KP_STAGES && !wait(&bar.v_empty[st], n / KP_STAGES - 1)) break;
        if (has_v) {
          uint8_t *tile = smem + H::V_OFF + st * H::V_HALF;
#pragma unroll
          for (int i = 0; i < VN; ++i) kp_store_codes(vr[i], tile, KP_BLOCK, vkey + i * VSTEP, vch);
        }
        publish(&bar.v_full[st]);
        if (has_v) load_v(id_v);
      }
      id_v = id_k;
      id_k = id_next;
    }
  } else {
    // ================================================== softmax, a thread per row
    kp_regs_inc<KP_R_SOFT>();
    const int hf = wg - 2, r = tid & 127, R = r_base + r;  // tiles hf, hf + 2, ...; S slot hf
    int vis;
    if constexpr (SEG)
      vis = row_at(R).vis;
    else
      vis = R < rows ? sp.visible(p.row_of(R)) : 0;
    const bool one = n_tiles == 1;
    const float shift = one ? KP_SHIFT_ONE : KP_SHIFT;
    float m = -INFINITY, l = 0.f, lvref = KP_NO_SCALE;
    // scales of the 16-key group lane % 8 of a tile: K scale (-1: no such page)
    // and log2 of the V scale, loaded two tiles ahead, page numbers four
    auto group_entry = [&](int t) {
      const int key = t * KP_KT + (lane & 7) * 16;
      return t < t1 && key < kend ? kv8_page_load(table, table_len, key >> p.shift) : -1;
    };
    auto group_scales = [&](int entry, float &ks, float &vs) {
      const bool there = (unsigned)entry < (unsigned)p.c.pages;
      ks = there ? __ldg(p.c.k_scales + (size_t)entry * p.c.kv_heads + h) : -1.f;
      vs = there ? __ldg(p.c.v_scales + (size_t)entry * p.c.kv_heads + h) : 0.f;
    };
    const int entry_0 = group_entry(t0 + hf);
    int entry_n = group_entry(t0 + hf + 2);
    // Queries: D / 8 lanes per row, f16 after the row's power of two. They come
    // through shared memory so that both loops can stay rolled: code that runs once
    // costs mostly its fetching.
    constexpr int LPR = D / 8, PASS = 256 / LPR;
    const int qtid = tid - 256, c8 = qtid % LPR;
    auto place = [&](int qr) {
      return reinterpret_cast<uint4 *>(smem + (c8 >> 3) * KP_BLOCK + kp_sw(qr, c8 & 7));
    };
    if (n_tiles > 0) {
#pragma unroll 2
      for (int qr = qtid / LPR; qr < 128; qr += PASS) {
        const Kv8SegRow x = row_at(r_base + qr);
        const uint16_t *src =
            p.q + x.b * p.qb + (int64_t)(h * p.rep + x.hr) * p.qh + (int64_t)x.i * p.ql + c8 * 8;
        const bool there = x.vis > 0;
        if (there && p.vec)
          cp_async16(place(qr), src);
        else
          *place(qr) = there ? kv8_load8(src, false) : make_uint4(0, 0, 0, 0);
      }
    }
    cp_async_commit();
    float ks_n, vs_n;
    group_scales(entry_0, ks_n, vs_n);
    ready();
    cp_async_wait<0>();
    if (n_tiles > 0) {
      // two neighbouring lanes take a row; magnitudes of bf16 compare as integers
      kp_soft_sync();
      const int qr = qtid >> 1, qh = qtid & 1;
      auto chunk = [&](int c) {  // c-th 8 elements of the lane's half row
        if (D > 64) c ^= qh << 2;  // (the two lanes in different banks)
        const int q8 = qh * (D / 16) + c;
        return reinterpret_cast<uint4 *>(smem + (q8 >> 3) * KP_BLOCK + kp_sw(qr, q8 & 7));
      };
      uint32_t mag = 0;
#pragma unroll 4
      for (int c = 0; c < D / 16; ++c) {
        const uint4 w = *chunk(c);
        mag = __vmaxu2(mag, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu),
                                     __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
      }
      mag = __vmaxu2(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
      const float pw = kv8_q_power(__uint_as_float(max(mag << 16, mag & 0xFFFF0000u)));
#pragma unroll 4
      for (int c = 0; c < D / 16; ++c) {
        uint4 w = *chunk(c);
        w = make_uint4(kv8_q_h2(w.x, pw), kv8_q_h2(w.y, pw), kv8_q_h2(w.z, pw), kv8_q_h2(w.w, pw));
        *chunk(c) = w;
      }
      if (qh == 0) s_fac[qr] = p.scale_log2 / pw;
      tc::fence_proxy_async_smem();
      kp_soft_sync();
      if (tid == 256) kp_arrive_leader(&bar.q_full);
    }
    const float fac = n_tiles > 0 ? s_fac[r] : 0.f;
    const uint32_t trow = tmem + (((uint32_t)(warp & 3) * 32u) << 16);
    // After a wait has given up, the tiles are gone through with what TMEM holds
    // and without further waits: the warpgroups hand over to each other in every
    // tile.
    bool ok = true;
    for (int n = hf; n < n_tiles; n += 2) {
      const int t = t0 + n;
      const float ks_l = ks_n, lv_l = vs_n > 0.f ? log2f(vs_n) : KP_NO_SCALE;
      group_scales(entry_n, ks_n, vs_n);
      entry_n = group_entry(t + 4);
      float lv_top = lv_l;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1)
        lv_top = fmaxf(lv_top, __shfl_xor_sync(0xffffffffu, lv_top, o));
      const uint32_t missing = __ballot_sync(0xffffffffu, ks_l < 0.f) & 0xFFu;
      // groups whose V scale is 0: their weights count for l alone
      const uint32_t blank = __ballot_sync(0xffffffffu, lv_l == KP_NO_SCALE) & 0xFFu & ~missing;

      const int slot = n % H::SLOTS;
      const uint32_t srow = trow + slot * 128;
      ok = ok && wait(&bar.s_full[slot], n / H::SLOTS);
      tc::tc_fence_after();
      // S is read twice, 32 columns at a time, rather than kept in registers, in
      // rolled loops: the roles' code together has to fit the instruction cache
      const int lim = vis - t * KP_KT;  // visible keys of this tile
      const bool masked = lim < KP_KT || missing;
      auto mask = [&](uint32_t (&v)[32], int c) {  // columns 32 c .. of the tile
        const int n = lim - 32 * c;
        uint32_t keep = n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
        if ((missing >> (2 * c)) & 1) keep &= 0xFFFF0000u;
        if ((missing >> (2 * c)) & 2) keep &= 0x0000FFFFu;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!((keep >> j) & 1)) v[j] = 0xFF800000u;
      };
      // K factor of a 16-key group; at least 2^-100, where z is 0 for any codes and a
      // masked score stays -inf (scale 0 makes every score of the page 0)
      const float kf_l = fmaxf(ks_l, 0.f);
      float fq = fac, least = 7.9e-31f;
      auto factor = [&](int g) { return fmaf(fq, __shfl_sync(0xffffffffu, kf_l, g), least); };
      float top = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32], w[32];
        tc::tmem_ld32(srow + c * 64, v);
        tc::tmem_ld32(srow + c * 64 + 32, w);
        tc::tmem_ld_wait();
        if (masked) { mask(v, 2 * c); mask(w, 2 * c + 1); }
#pragma unroll
        for (int gg = 0; gg < 4; ++gg) {
          const uint32_t *u = (gg & 2 ? w : v) + (gg & 1) * 16;
          float x0 = kp_max3(u[0], u[1], u[2]), x1 = kp_max3(u[3], u[4], u[5]);
          float x2 = kp_max3(u[6], u[7], u[8]), x3 = kp_max3(u[9], u[10], u[11]);
          x0 = kp_max3(__float_as_uint(x0), u[12], u[13]);
          x1 = kp_max3(__float_as_uint(x1), u[14], u[15]);
          top = fmaxf(top, fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * factor(4 * c + gg));
        }
      }
      // maximum and v after the tile before this one, and after this one
      float m_prev = -INFINITY, lv_prev = KP_NO_SCALE;
      if (n > 0) {
        kp_take_over(hf ^ 1);
        m_prev = s_m[r];
        lv_prev = s_lv[hf ^ 1];
      }
      const bool move = top > __fadd_rd(m_prev, KP_SHIFT + KP_MOVE);
      const float m_new = move ? __fadd_ru(top, -shift) : m_prev;
      lvref = one ? lv_top : fmaxf(lv_prev, ceilf(lv_top));
      s_m[r] = m_new;
      if (r == 0) s_lv[hf] = lvref;
      if (n + 1 < n_tiles) kp_hand_over(hf);
      l *= kp_ratio(m, m_new);  // (the other warpgroup may have moved it too)
      m = m_new;
      if (ok && n > 0 && (lvref > lv_prev || __any_sync(0xffffffffu, move))) {  // rescale O
        ok = wait(&bar.o_done[(n - 1) % H::SLOTS], (n - 1) / H::SLOTS);
        tc::tc_fence_after();
        const float a = kp_ratio(m_prev, m_new) * kp_ex2(lv_prev - lvref);
        if (ok) {
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t v[32];
            tc::tmem_ld32(trow + H::O_COL + c0, v);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
            kp_tmem_st32(trow + H::O_COL + c0, v);
          }
          kp_tmem_st_wait();
        }
      }
      float sub = m == -INFINITY ? 0.f : -m;
      // Scores so large that a product, which z - m takes unrounded below, may lie whole
      // powers of two off the rounded maximum: the row's S becomes z - m first, rounded
      // alike.
      const bool large = fabsf(sub) > 65536.f;
      if (__any_sync(0xffffffffu, large)) {
#pragma unroll 1
        for (int g = 0; g < 8; ++g) {
          const float f = factor(g);
          uint32_t v[16];
          tc::tmem_ld16(srow + g * 16, v);
          tc::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (large) v[j] = __float_as_uint(__fadd_rn(__fmul_rn(__uint_as_float(v[j]), f), sub));
          kp_tmem_st16(srow + g * 16, v);
        }
        kp_tmem_st_wait();
        if (large) {
          sub = fq = 0.f;
          least = 1.f;
        }
      }
      // log2 of V scale / v of the lane's group, and the way back for l: bounded, so that
      // exponentials whose weight rounds to 0 in f16 are there for l
      const float cg_l = lv_l > KP_NO_SCALE ? fmaxf(lv_l - lvref, -60.f) : 0.f;
      const float back_l = kp_ex2(-cg_l);
      // (P, 16 columns, only goes over columns that have been read)
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32], pk[16];
        tc::tmem_ld32(srow + c * 32, v);
        tc::tmem_ld_wait();
        if (masked) mask(v, c);
#pragma unroll
        for (int gg = 0; gg < 2; ++gg) {
          const int g = 2 * c + gg;
          const float f = factor(g), cg = __fadd_rd(sub, __shfl_sync(0xffffffffu, cg_l, g));
          const float back = __shfl_sync(0xffffffffu, back_l, g);
          const f2 ff = f2_make(f, f), cc = f2_make(cg, cg);
          float e[16];
#pragma unroll
          for (int j = 0; j < 16; j += 2)
            f2_split(f2_fma(f2_make(__uint_as_float(v[gg * 16 + j]),
                                    __uint_as_float(v[gg * 16 + j + 1])), ff, cc),
                     e[j], e[j + 1]);
#pragma unroll
          for (int j = 0; j < 16; ++j) e[j] = kp_ex2(e[j]);
          f2 sum0 = f2_make(e[0], e[1]), sum1 = f2_make(e[2], e[3]);
#pragma unroll
          for (int j = 4; j < 16; j += 4) {
            sum0 = f2_add(sum0, f2_make(e[j], e[j + 1]));
            sum1 = f2_add(sum1, f2_make(e[j + 2], e[j + 3]));
          }
          float s0, s1;
          f2_split(f2_add(sum0, sum1), s0, s1);
          l = fmaf(s0 + s1, back, l);
#pragma unroll
          for (int j = 0; j < 16; j += 2) pk[gg * 8 + (j >> 1)] = pack_h2(e[j], e[j + 1]);
        }
        kp_tmem_st16(srow + c * 16, pk);
      }
      kp_tmem_st_wait();
      if (blank) {  // (rare, so the weights are first written as if they counted)
#pragma unroll 1
        for (int g = 0; g < 8; ++g)
          if ((blank >> g) & 1) kp_tmem_zero8(srow + g * 8);
        kp_tmem_st_wait();
      }
      tc::tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) kp_arrive_leader(&bar.p_full[slot]);
    }
    // ---- the row's m, v and l after the last tile, and its O after the last product
    kp_soft_sync();
    if (n_tiles > 0) {
      const float m_end = s_m[r];
      l *= kp_ratio(m, m_end);
      m = m_end;
      lvref = s_lv[(n_tiles - 1) & 1];
    }
    s_l[hf][r] = l;
    kp_soft_sync();
    l = s_l[0][r] + s_l[1][r];
    if (ok && n_tiles > 0) {
      ok = wait(&bar.o_last, 0);
      tc::tc_fence_after();
    }
    if (ok) {
      const float v = kp_ex2(lvref);
      const int i = p.row_of(R), hr = R - i * p.rep, r_pair = rank * 128 + r;
      const size_t row = ((size_t)b * p.Hq + h * p.rep + hr) * p.L + i;
      const bool live = R < rows;
      if (live && hf == 0) {
        if (SEG || p.splits > 1)
          p.ml_part[tile_id * KP_ROWS + r_pair] = make_float2(m, l);
        else if (p.lse)
          p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
      }
      // the warp's 32 rows x 32 dims go through the queries' place, which no product
      // reads any more, so that a store covers whole 64-byte pieces of 8 rows
      uint8_t *turn = smem + (warp - 8) * 2048;
      const float inv = SEG || p.splits > 1 ? v : l == 0.f ? 0.f : v / l;
#pragma unroll 1
      for (int c0 = hf * (D / 2); c0 < (hf + 1) * (D / 2); c0 += 32) {
        uint32_t x[32];
        if (n_tiles > 0) {
          tc::tmem_ld32(trow + H::O_COL + c0, x);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = 0;
        }
        float y[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) y[j] = __uint_as_float(x[j]) * inv;
        __syncwarp();
        if (SEG || p.splits > 1) {
          if (live && n_tiles > 0) {
            float *d = p.o_part + (tile_id * KP_ROWS + r_pair) * D + c0;
#pragma unroll
            for (int q = 0; q < 32; q += 8) kp_store32(d + q, y + q);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(turn + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) =
                make_uint4(pack_bf2(y[8 * q], y[8 * q + 1]), pack_bf2(y[8 * q + 2], y[8 * q + 3]),
                           pack_bf2(y[8 * q + 4], y[8 * q + 5]),
                           pack_bf2(y[8 * q + 6], y[8 * q + 7]));
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int s = k * 8 + (lane >> 2), q = lane & 3;
            const uint32_t srow = __shfl_sync(0xffffffffu, live ? (uint32_t)row : 0xFFFFFFFFu, s);
            const uint4 x4 =
                *reinterpret_cast<const uint4 *>(turn + s * 64 + ((q ^ (s >> 1 & 3)) << 4));
            if (srow != 0xFFFFFFFFu)
              *reinterpret_cast<uint4 *>(p.out + (size_t)srow * D + c0 + q * 8) = x4;
          }
        }
        __syncwarp();
      }
    }
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

template <int D, bool SEG>
int kp_launch(const Kv8AttnParams &p, cudaStream_t s) {
  using H = KpShape<D>;
  static std::atomic<uint64_t> ready{0};
  const int rc = once_per_device(ready, [] {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kv8_prefill_kernel<D, SEG>);
    // the warpgroups' register shares add up to 128 per thread at launch
    if (e == cudaSuccess && fa.numRegs != 128)
      return set_error(VB_ERR_CUDA, "kv8_prefill_kernel: built with %d registers, 128 needed",
                       fa.numRegs);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kv8_prefill_kernel<D, SEG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               H::SMEM);
    return e == cudaSuccess ? VB_OK
                            : set_error(VB_ERR_CUDA, "kv8_prefill_kernel attributes: %s",
                                        cudaGetErrorString(e));
  });
  if (rc != VB_OK) return rc;
  const unsigned pairs = SEG ? p.pairs : p.row_tiles * p.splits * p.c.kv_heads * p.c.batch;
  vb_launch(kv8_prefill_kernel<D, SEG>, dim3(2 * pairs), dim3(KP_THREADS), H::SMEM, s, false, p);
  return check_launch("kv8_prefill_kernel");
}

}  // namespace

int kv8_prefill_rows() { return KP_ROWS; }

int kv8_prefill_launch(const Kv8AttnParams &p, cudaStream_t s) {
  switch (p.c.dim) {
    case 64: return kp_launch<64, false>(p, s);
    case 128: return kp_launch<128, false>(p, s);
    default: return kp_launch<256, false>(p, s);
  }
}

int kv8_prefill_launch_segments(const Kv8AttnParams &p, cudaStream_t s) {
  switch (p.c.dim) {
    case 64: return kp_launch<64, true>(p, s);
    case 128: return kp_launch<128, true>(p, s);
    default: return kp_launch<256, true>(p, s);
  }
}

}  // namespace vb
