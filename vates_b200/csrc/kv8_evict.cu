// Eviction from the paged 8-bit cache: of every sequence that holds more than
// `keep` rows, each kv head keeps the ones with the largest weight.
//
// Rows of one (sequence, kv head) are ordered by (protected, weight, lower row):
// protected are the rows below `first` and those whose position is above
// newest - recent. The best `keep` stay. The evicted rows below `keep` are holes,
// and the j-th hole takes the j-th kept row from `keep` on, so only as many rows
// move as are evicted below `keep`: a sequence that is a few rows over its share
// moves a few rows, not all behind the first hole. (Attention does not care in
// which row a key lies.) A page that receives rows takes the largest scale among
// the pages that its live rows come from, s; codes become rint(code * (from / s)),
// which leaves the rows of that page as they are.
//
// kv8_evict_select_kernel: a cluster of up to 8 CTAs owns one (sequence, kv head).
// Weights become 32-bit keys in their order (kept in shared memory); up to three
// histograms of 11, 11 and 10 bits give the last key that stays: every CTA adds the
// bins that it has rows in to those of all others (reading all bins of all others
// instead took 5 us of 20 for 65,536 rows). Ballots count and number holes and
// moving rows, in order.
// kv8_evict_move_kernel: groups of 32 to 128 threads fill the holes of one page of K or
// V after another, and move weights and positions with K. Nothing is written that
// another group still reads: rows move from `keep` on to below it, and the scale of the
// page in which `keep` falls is taken down by the first kernel.
//
// What bounds it: latency, of a dozen steps that each need the one before. 2 heads with
// 4,160 rows of 256 down to 4,096 take 13.5 us, of which the selection 9; 256 heads with up
// to 2,111 rows of 128 down to 2,048 23 us (45 where every second page has to take a larger
// scale); 4 heads with 65,536 rows of 256 down to 8,192 20 (37).
#include "kv8.cuh"

namespace vb {
namespace {

constexpr int EV_CTAS = 8;            // most CTAs of a cluster
constexpr int EV_BINS = 2048;
constexpr int EV_HELD = 16;           // rows that a thread holds the keys of
constexpr int EV_KEYS = 24576;        // else: most keys of a CTA in shared memory
constexpr uint32_t EV_SAFE = 0xFFFFFFFFu;

struct Kv8EvictParams {
  VbKv8Cache c;
  float *weights;
  int32_t *positions;
  const int32_t *lens;
  int32_t *lens_out;
  int32_t *status;
  // per (sequence, head): holes, moving rows, first hole of a page, and the K and V scale
  // of the page in which `keep` falls
  int32_t *lists;
  long long list_stride;
  int most;                  // room of a list
  int room, cap, keep, first, recent, shift, cached;
};

__device__ __forceinline__ uint32_t ev_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t ev_ctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// All threads of the cluster meet; what they wrote to shared memory is visible.
__device__ __forceinline__ void ev_sync(uint32_t ctas) {
  if (ctas == 1)
    __syncthreads();
  else
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
}
// Adds to a word of CTA `rank`'s shared memory.
__device__ __forceinline__ void ev_peer_add(uint32_t *p, uint32_t rank, uint32_t x) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(x) : "memory");
}
// A word of CTA `rank`'s shared memory. (Not ordered among themselves, so that several are
// on their way at once; the barriers around them are.)
__device__ __forceinline__ uint32_t ev_peer(const void *p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}

// HELD: a thread has up to EV_HELD rows, whose keys stay in registers (each pass over
// the rows costs instructions more than anything else); else keys are in shared memory,
// up to p.cached of them.
template <int EV_THREADS, bool HELD>
__global__ void __launch_bounds__(EV_THREADS) kv8_evict_select_kernel(const __grid_constant__ Kv8EvictParams p) {
  constexpr int EV_WARPS = EV_THREADS / 32, EV_PER = EV_BINS / EV_THREADS;
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[EV_BINS], s_all[3][EV_BINS];  // the CTA's; the cluster's
  __shared__ uint32_t s_warp[2][EV_WARPS], s_total[3];  // total: ties; holes, moving rows
  __shared__ uint32_t s_bin, s_above, s_count;
  __shared__ int s_newest;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = ev_rank(), C = ev_ctas();
  const int unit = blockIdx.x / C, b = unit / p.c.kv_heads, h = unit % p.c.kv_heads;
  const int len = p.lens[b], n = min(max(len, 0), p.cap);
  if (rank == 0 && h == 0 && tid == 0) {
    if (len != n) flag_status(p.status, VB_STATUS_BOUNDS);
    p.lens_out[b] = min(n, p.keep);
  }
  if (n <= p.keep) return;  // (every CTA of the cluster)
  float *weights = p.weights + (size_t)unit * p.room;
  int32_t *positions = p.positions ? p.positions + (size_t)unit * p.room : nullptr;
  int32_t *holes = p.lists + unit * p.list_stride, *moving = holes + p.most,
          *firsts = moving + p.most;
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
  // the CTA's rows, and this warp's 32 * turns of them
  const int turns = (int)((n + (long long)C * EV_THREADS - 1) / ((long long)C * EV_THREADS));
  const int at0 = warp * turns * 32 + lane, row0 = (int)rank * EV_THREADS * turns + at0;

  auto order = [&](float w) {
    w += 0.f;  // (-0 is 0)
    const uint32_t k = __float_as_uint(w);
    return w != w ? 0u : k >> 31 ? ~k : k | 0x80000000u;
  };
  for (int i = tid; i < EV_BINS; i += EV_THREADS)
    s_hist[i] = s_all[0][i] = s_all[1][i] = s_all[2][i] = 0;
  // Goes through the warp's rows: f(turn, row number).
  auto rows = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int t = 0; t < EV_HELD; ++t)
        if (t < turns) f(t, row0 + t * 32);
    } else {
      for (int t = 0; t < turns; ++t) f(t, row0 + t * 32);
    }
  };
  // ---- the weights' order, and the newest position
  const bool dated = p.recent > 0 && positions;
  int newest = -0x7fffffff - 1;
  uint32_t held[HELD ? EV_HELD : 1];
  int date[HELD ? EV_HELD : 1];
  if constexpr (HELD) {
    rows([&](int t, int i) {
      held[t] = __float_as_uint(i < n ? weights[i] : 0.f);
      date[t] = !dated ? i : i < n ? positions[i] : newest;
    });
    rows([&](int t, int i) {
      held[t] = order(__uint_as_float(held[t]));
      if (dated) newest = max(newest, date[t]);
    });
  } else {
    for (int t0 = 0; t0 < turns; t0 += 4) {
      float w[4];
      int q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = row0 + (t0 + k) * 32, at = at0 + (t0 + k) * 32;
        const bool there = t0 + k < turns && i < n;
        w[k] = there && at < p.cached ? weights[i] : 0.f;
        q[k] = there && dated ? positions[i] : newest;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int at = at0 + (t0 + k) * 32;
        newest = max(newest, q[k]);
        if (t0 + k < turns && at < p.cached) s_keys[at] = order(w[k]);
      }
    }
  }
  if (dated) {
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) s_warp[0][warp] = (uint32_t)newest;
    __syncthreads();
    if (warp == 0) {
      newest = __reduce_max_sync(0xffffffffu, (int)s_warp[0][lane % EV_WARPS]);
      if (lane == 0) s_newest = newest;
    }
  }
  ev_sync(C);  // (and all bins are zero)
  if (dated) {
    newest = (int)ev_peer(&s_newest, min((uint32_t)lane, C - 1));
    newest = __reduce_max_sync(0xffffffffu, newest);
  } else {
    newest = n - 1;
  }
  // positions above it are protected
  const long long late = p.recent > 0 ? (long long)newest - p.recent : 0x7fffffffffffll;
  if constexpr (HELD) {
    rows([&](int t, int i) {
      if (i < p.first || date[t] > late) held[t] = EV_SAFE;
    });
  } else {
    rows([&](int t, int i) {
      const int at = at0 + t * 32;
      if (at < p.cached && (i < p.first || (dated && i < n ? positions[i] : i) > late))
        s_keys[at] = EV_SAFE;
    });
  }
  auto key = [&](int t, int i) {
    if constexpr (HELD) {
      return held[t];
    } else {
      const int at = at0 + t * 32;
      if (at < p.cached) return s_keys[at];
      return i < p.first || (dated ? positions[i] : i) > late ? EV_SAFE : order(weights[i]);
    }
  };

  // ---- the key of the last row that stays: `need` of the rows that have it do
  uint32_t last = 0, prefix = 0, need = (uint32_t)p.keep;
  bool ties = true;  // not all rows with the last key stay: the lower ones
#pragma unroll 1
  for (int d = 0; d < 3 && ties; ++d) {
    const int low = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
    if (d > 0 && C > 1) {
      for (int i = tid; i < EV_BINS; i += EV_THREADS) s_hist[i] = 0;
      __syncthreads();
    }
    uint32_t *hist = C > 1 ? s_hist : s_all[d];
    rows([&](int t, int i) {
      if (i >= n) return;
      const uint32_t k = key(t, i);
      if (d == 0 || k >> (low + bits) == prefix)
        atomicAdd(hist + ((k >> low) & ((1u << bits) - 1)), 1u);
    });
    __syncthreads();
    if (C > 1) {
      for (int i = tid; i < EV_BINS; i += EV_THREADS) {
        const uint32_t x = s_hist[i];
        if (x)
          for (uint32_t r = 0; r < C; ++r) ev_peer_add(s_all[d] + i, r, x);
      }
      ev_sync(C);
    }
    // bins from the top: thread tid has EV_PER of them from EV_BINS - 1 - EV_PER tid down
    uint32_t bin[EV_PER], mine = 0;
#pragma unroll
    for (int x = 0; x < EV_PER; ++x) bin[x] = s_all[d][EV_BINS - 1 - EV_PER * tid - x];
#pragma unroll
    for (int x = 0; x < EV_PER; ++x) mine += bin[x];
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_warp[0][warp] = inc;
    __syncthreads();
    uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[0][lane] : 0u);
    before += inc - mine;
#pragma unroll
    for (int x = 0; x < EV_PER; ++x) {
      if (before < need && need <= before + bin[x]) {
        s_bin = EV_BINS - 1 - EV_PER * tid - x;
        s_above = before;
        s_count = bin[x];
      }
      before += bin[x];
    }
    __syncthreads();
    need -= s_above;
    prefix = prefix << bits | s_bin;
    last = prefix << low;
    ties = need < s_count;  // all rows of the bin stay: no need to look closer
    __syncthreads();  // s_warp, s_bin are free again
  }

  // Exclusive sums over the warps and CTAs before this warp of up to two counts.
  auto before = [&](uint32_t a, uint32_t c, int slot, uint32_t &sa, uint32_t &sc) {
    if (lane == 0) {
      s_warp[0][warp] = a;
      s_warp[1][warp] = c;
    }
    __syncthreads();
    const uint32_t ta = lane < EV_WARPS ? s_warp[0][lane] : 0u;
    const uint32_t tc = lane < EV_WARPS ? s_warp[1][lane] : 0u;
    sa = __reduce_add_sync(0xffffffffu, lane < warp ? ta : 0u);
    sc = __reduce_add_sync(0xffffffffu, lane < warp ? tc : 0u);
    if (warp == 0) {
      const uint32_t all_a = __reduce_add_sync(0xffffffffu, ta);
      const uint32_t all_c = __reduce_add_sync(0xffffffffu, tc);
      if (lane == 0) {
        s_total[slot] = all_a;
        if (slot) s_total[2] = all_c;
      }
    }
    ev_sync(C);
    if (rank > 0) {
      const uint32_t r = min((uint32_t)lane, rank - 1);
      const uint32_t pa = ev_peer(s_total + slot, r), pc = ev_peer(s_total + (slot ? 2 : 0), r);
      sa += __reduce_add_sync(0xffffffffu, lane < rank ? pa : 0u);
      sc += __reduce_add_sync(0xffffffffu, lane < rank ? pc : 0u);
    }
  };
  uint32_t tie0 = 0, unused;
  if (ties) {
    uint32_t mine = 0;
    rows([&](int t, int i) {
      mine += __popc(__ballot_sync(0xffffffffu, i < n && key(t, i) == last));
    });
    before(mine, 0, 0, tie0, unused);
  }
  const uint32_t below = (1u << lane) - 1;
  // whether a row stays; `tie`: rows with the last key before this turn
  auto stays = [&](int t, int i, uint32_t &tie) {
    const uint32_t k = i < n ? key(t, i) : 0u;
    if (!ties) return i < n && k >= last;
    const uint32_t same = __ballot_sync(0xffffffffu, i < n && k == last);
    const bool s = i < n && (k > last || (k == last && tie + __popc(same & below) < need));
    tie += __popc(same);
    return s;
  };
  uint32_t n_holes = 0, n_moving = 0, tie = tie0;
  rows([&](int t, int i) {
    const bool s = stays(t, i, tie);
    n_holes += __popc(__ballot_sync(0xffffffffu, !s && i < p.keep));
    n_moving += __popc(__ballot_sync(0xffffffffu, s && i >= p.keep));
  });
  uint32_t hole, move;
  before(n_holes, n_moving, 1, hole, move);
  tie = tie0;
  rows([&](int t, int i) {
    const bool s = stays(t, i, tie);
    const uint32_t hb = __ballot_sync(0xffffffffu, !s && i < p.keep);
    const uint32_t mb = __ballot_sync(0xffffffffu, s && i >= p.keep);
    if (i < p.keep) {
      const uint32_t at = hole + __popc(hb & below), mine = (hb >> lane) & 1;
      if ((i & (p.c.page - 1)) == 0) firsts[i >> p.shift] = (int)at;
      if (i == p.keep - 1)  // the number of holes, behind the last page
        firsts[(p.keep + p.c.page - 1) >> p.shift] = (int)(at + mine);
      if (mine) holes[at] = i;
    }
    if ((mb >> lane) & 1) moving[move + __popc(mb & below)] = i;
    hole += __popc(hb);
    move += __popc(mb);
  });
  // the page in which `keep` falls: rows of it may move, and its scale may change
  if (rank == 0 && tid < 2) {
    const int id = kv8_page(table, p.c.max_pages, p.c.pages, p.keep >> p.shift, nullptr);
    const float *scales = tid ? p.c.v_scales : p.c.k_scales;
    firsts[((p.keep + p.c.page - 1) >> p.shift) + 1 + tid] =
        id < 0 ? 0 : __float_as_int(scales[(size_t)id * p.c.kv_heads + h]);
  }
  if (C > 1) ev_sync(C);  // no CTA ends while another may still read its shared memory
}

constexpr int EM_THREADS = 256;
constexpr int EM_AHEAD = 4;   // pieces of 16 codes that a thread has in flight

// G: threads for a page of K or of V, no fewer than it has rows.
template <int G>
__global__ void __launch_bounds__(EM_THREADS, 4) kv8_evict_move_kernel(const __grid_constant__ Kv8EvictParams p) {
  constexpr int GROUPS = EM_THREADS / G, SLOTS = GROUPS / 2, WARPS = G / 32;
  __shared__ int s_src[GROUPS][G], s_sid[GROUPS][G], s_row[GROUPS][G];
  __shared__ float s_from[GROUPS][G], s_top[GROUPS][WARPS];
  __shared__ uint32_t s_filled[GROUPS][4][WARPS];
  __shared__ int s_moved[GROUPS][WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int gi = threadIdx.x / G, kv = gi & 1, tid = threadIdx.x % G, warp = tid >> 5;
  const int lane = tid & 31, unit = blockIdx.x, b = unit / p.c.kv_heads, h = unit - b * p.c.kv_heads;
  if (p.lens[b] <= p.keep) return;
  const int pages = (p.keep + p.c.page - 1) >> p.shift, edge = p.keep >> p.shift;
  const int32_t *holes = p.lists + unit * p.list_stride, *moving = holes + p.most,
                *firsts = moving + p.most;
  const float edge_scale = __int_as_float(firsts[pages + 1 + kv]);
  const int32_t *table = p.c.page_table + (size_t)b * p.c.max_pages;
  const int D = p.c.dim, lpr = D >> 4, lsh = D == 64 ? 2 : D == 128 ? 3 : 4;
  const size_t page_bytes = (size_t)p.c.page * D;
  int8_t *codes = kv ? p.c.v_codes : p.c.k_codes;
  float *scales = kv ? p.c.v_scales : p.c.k_scales;
  auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + gi), "n"(G) : "memory"); };

  // the group's pages, 32 at a time: their first hole and the number of holes
  const int stride = gridDim.y * SLOTS;
  for (int pg0 = blockIdx.y * SLOTS + (gi >> 1); pg0 < pages; pg0 += 32 * stride) {
    const int mine = pg0 + lane * stride;
    int first_l = 0, count_l = 0;
    if (mine < pages) {
      first_l = firsts[mine];
      count_l = firsts[mine + 1] - first_l;
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, count_l > 0); todo; todo &= todo - 1) {
      const int at = __ffs(todo) - 1, pg = pg0 + at * stride;
      const int j0 = __shfl_sync(0xffffffffu, first_l, at);
      const int count = __shfl_sync(0xffffffffu, count_l, at);
      const int id = kv8_page(table, p.c.max_pages, p.c.pages, pg, tid == 0 ? p.status : nullptr);
      if (id < 0) continue;
      const int live = min(p.c.page, p.keep - (pg << p.shift));
      const float old = pg == edge ? edge_scale : scales[(size_t)id * p.c.kv_heads + h];
      // ---- hole `tid` of the page, and where its new row comes from; from a page that is
      // not there none does, and the hole's own row stays
      int src = -1, sid = -1, row = 0;
      float from = 0.f;
      if (tid < count) {
        src = moving[j0 + tid];
        row = holes[j0 + tid];
        sid = kv8_page(table, p.c.max_pages, p.c.pages, src >> p.shift, p.status);
        if (sid >= 0)
          from = (src >> p.shift) == edge ? edge_scale : scales[(size_t)sid * p.c.kv_heads + h];
        s_src[gi][tid] = src & (p.c.page - 1);
        s_sid[gi][tid] = sid;
        s_row[gi][tid] = row & (p.c.page - 1);
        s_from[gi][tid] = from;
        if (kv == 0 && sid >= 0) {
          const size_t w = (size_t)unit * p.room;
          p.weights[w + row] = p.weights[w + src];
          if (p.positions) p.positions[w + row] = p.positions[w + src];
        }
      }
      const int r = row & (p.c.page - 1);
      float top = from;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t f = __reduce_or_sync(0xffffffffu, sid >= 0 && r >> 5 == w ? 1u << (r & 31) : 0u);
        if (lane == 0) s_filled[gi][w][warp] = f;
      }
      const uint32_t all = __ballot_sync(0xffffffffu, sid >= 0);
      if (lane == 0) {
        s_top[gi][warp] = top;
        s_moved[gi][warp] = __popc(all);
      }
      meet();
      int moved = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) moved += s_moved[gi][w];
      const bool stay = moved < live;
      top = stay ? old : 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_top[gi][w]);

      // ---- rows that move, and rows that stay but take a larger scale
      uint4 *dst = reinterpret_cast<uint4 *>(codes + ((size_t)id * p.c.kv_heads + h) * page_bytes);
      for (int x0 = tid; x0 < count << lsh; x0 += G * EM_AHEAD) {
        uint4 v[EM_AHEAD];
#pragma unroll
        for (int k = 0; k < EM_AHEAD; ++k) {
          const int x = x0 + k * G, o = x >> lsh;
          if (o < count && s_sid[gi][o] >= 0)
            v[k] = reinterpret_cast<const uint4 *>(
                codes + ((size_t)s_sid[gi][o] * p.c.kv_heads + h) * page_bytes)[
                (s_src[gi][o] << lsh) + (x & (lpr - 1))];
        }
#pragma unroll
        for (int k = 0; k < EM_AHEAD; ++k) {
          const int x = x0 + k * G, o = x >> lsh;
          if (o < count && s_sid[gi][o] >= 0) {
            const float ratio = top > 0.f ? __fdiv_rn(s_from[gi][o], top) : 1.f;
            dst[(s_row[gi][o] << lsh) + (x & (lpr - 1))] = ratio == 1.f ? v[k] : kv8_recode(v[k], ratio);
          }
        }
      }
      if (stay && top > old) {
        const float ratio = __fdiv_rn(old, top);
        uint32_t filled[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          filled[w] = 0;
#pragma unroll
          for (int x = 0; x < WARPS; ++x) filled[w] |= s_filled[gi][w][x];
        }
        auto stays = [&](int x) {
          const int y = x >> lsh;
          const uint32_t f = y < 64 ? (y < 32 ? filled[0] : filled[1]) : (y < 96 ? filled[2] : filled[3]);
          return y < live && !((f >> (y & 31)) & 1);
        };
        for (int x0 = tid; x0 < live << lsh; x0 += G * EM_AHEAD) {
          uint4 v[EM_AHEAD];
#pragma unroll
          for (int k = 0; k < EM_AHEAD; ++k)
            if (stays(x0 + k * G)) v[k] = dst[x0 + k * G];
#pragma unroll
          for (int k = 0; k < EM_AHEAD; ++k)
            if (stays(x0 + k * G)) dst[x0 + k * G] = kv8_recode(v[k], ratio);
        }
      }
      if (tid == 0 && top != old) scales[(size_t)id * p.c.kv_heads + h] = top;
      meet();  // the page's holes have been read
    }
  }
}

struct EvictPlan {
  int cap, most, threads, ctas, cached;
  bool held;
  long long stride;
  size_t bytes;
};

// Rows beyond what the table and the weights have room for do not exist; up to
// min(keep, cap - keep) rows move.
EvictPlan ev_plan(const VbKv8EvictArgs *a) {
  EvictPlan pl;
  const long long rows = (long long)a->cache.max_pages * a->cache.page;
  pl.cap = (int)(rows < a->room ? rows : a->room);
  const int over = pl.cap > a->keep ? pl.cap - a->keep : 0;
  pl.most = over < a->keep ? over : a->keep;
  const long long units = (long long)a->cache.batch * a->cache.kv_heads;
  // Up to 8 rows a thread, then more CTAs, as long as every one of 1024 threads has an SM
  // (4,160 rows of 2 heads: one CTA a head 8.7 us, four 12: each barrier of a cluster
  // costs half a microsecond, a row of a thread 0.6 in all).
  pl.threads = units <= 148 ? 1024 : 512;
  pl.ctas = 1;
  while (pl.ctas < EV_CTAS && units * pl.ctas * 2 <= 148 && pl.cap > 8 * pl.threads * pl.ctas)
    pl.ctas *= 2;
  const long long per = align_up((pl.cap + pl.ctas - 1) / pl.ctas, pl.threads);
  pl.held = per <= EV_HELD * pl.threads;
  pl.cached = (int)(pl.held ? 0 : per < EV_KEYS ? per : EV_KEYS);
  pl.stride = 2ll * pl.most + ((long long)a->keep + a->cache.page - 1) / a->cache.page + 3;
  pl.bytes = pl.most ? (size_t)(units * pl.stride) * sizeof(int32_t) : 0;
  return pl;
}

template <int T, bool HELD>
int ev_select(const Kv8EvictParams &p, const EvictPlan &pl, long long units, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  const int set = once_per_device(ready, [] {
    const cudaError_t e = cudaFuncSetAttribute(
        kv8_evict_select_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_KEYS * 4);
    return e == cudaSuccess ? VB_OK
                            : set_error(VB_ERR_CUDA, "kv8_evict_select_kernel attributes: %s",
                                        cudaGetErrorString(e));
  });
  if (set != VB_OK) return set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * pl.ctas));
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = (size_t)pl.cached * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pl.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kv8_evict_select_kernel<T, HELD>, p);
  return check_launch("kv8_evict_select_kernel");
}

int ev_check(const VbKv8EvictArgs *a) {
  VB_REQUIRE(a, "vb_kv8_evict: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_evict");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->keep >= 1 && a->room >= 0 && a->room <= 0x7fffffff - 65536,
             "vb_kv8_evict: keep=%d room=%d", a->keep, a->room);
  VB_REQUIRE((long long)a->cache.batch * a->cache.kv_heads <= 1 << 28,
             "vb_kv8_evict: %d sequences of %d kv heads", a->cache.batch, a->cache.kv_heads);
  VB_REQUIRE(a->first >= 0 && a->recent >= 0 && (long long)a->first + a->recent <= a->keep,
             "vb_kv8_evict: first=%d recent=%d of keep=%d", a->first, a->recent, a->keep);
  return VB_OK;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

size_t vb_kv8_evict_workspace_size(const VbKv8EvictArgs *a) {
  return ev_check(a) == VB_OK ? ev_plan(a).bytes : 0;
}

int vb_kv8_evict(const VbKv8EvictArgs *a, vb_stream_t stream) {
  const int rc = ev_check(a);
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->lens && a->lens_out && a->lens != a->lens_out, "vb_kv8_evict: lens and lens_out");
  VB_REQUIRE(a->weights || a->room == 0, "vb_kv8_evict: null weights");
  const EvictPlan pl = ev_plan(a);
  if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes))
    return set_error(VB_ERR_WORKSPACE, "vb_kv8_evict: workspace %zu < %zu bytes",
                     a->workspace_bytes, pl.bytes);
  VB_REQUIRE(((uintptr_t)a->workspace % 16) == 0, "vb_kv8_evict: workspace alignment");
  const long long units = (long long)a->cache.batch * a->cache.kv_heads;
  Kv8EvictParams p;
  p.c = a->cache;
  p.weights = a->weights; p.positions = a->positions;
  p.lens = a->lens; p.lens_out = a->lens_out; p.status = a->status;
  p.lists = static_cast<int32_t *>(a->workspace);
  p.list_stride = pl.stride; p.most = pl.most;
  p.room = a->room; p.cap = pl.cap; p.keep = a->keep; p.first = a->first; p.recent = a->recent;
  p.shift = kv8_page_shift(a->cache.page);
  p.cached = pl.cached;
  cudaStream_t s = as_stream(stream);
  const int rc2 = pl.threads == 1024 ? (pl.held ? ev_select<1024, true>(p, pl, units, s)
                                                : ev_select<1024, false>(p, pl, units, s))
                                     : (pl.held ? ev_select<512, true>(p, pl, units, s)
                                                : ev_select<512, false>(p, pl, units, s));
  if (rc2 != VB_OK || pl.most == 0) return rc2;
  // Threads for a page: up to eight pieces of 16 codes each, and no fewer than rows.
  const int pages = (a->keep + a->cache.page - 1) / a->cache.page;
  const int pieces = a->cache.page * a->cache.dim / 16, page = a->cache.page;
  const int group = page <= 32 && pieces <= 256 ? 32 : page <= 64 && pieces <= 512 ? 64 : 128;
  // CTAs of a (sequence, head): enough for all pages, fewer once that fills the SMs several
  // times
  const int per = EM_THREADS / (2 * group), want = (pages + per - 1) / per;
  const long long few = (148 * 16 + units - 1) / units;
  const dim3 grid((unsigned)units, (unsigned)(want < few ? want : few)), block(EM_THREADS);
  if (group == 32) vb_launch(kv8_evict_move_kernel<32>, grid, block, 0, s, true, p);
  else if (group == 64) vb_launch(kv8_evict_move_kernel<64>, grid, block, 0, s, true, p);
  else vb_launch(kv8_evict_move_kernel<128>, grid, block, 0, s, true, p);
  return check_launch("kv8_evict_move_kernel");
}

}  // extern "C"
