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
// A cluster of up to 8 CTAs owns one (sequence, kv head). Weights become 32-bit
// keys in their order (kept in shared memory); three histograms of 11, 11 and 10
// bits, added up over the cluster, give the last key that stays. Ballots count
// and number holes and moving rows, in order, and then a warp takes a page of K
// or V at a time.
// Nothing is written that another warp still reads: rows move from `keep` on to
// below it, and the scale of the page in which `keep` falls is read beforehand.
#include "kv8.cuh"

namespace vb {
namespace {

constexpr int EV_THREADS = 1024;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_KEYS = 24576;        // most keys of a CTA in shared memory
constexpr uint32_t EV_SAFE = 0xFFFFFFFFu;

struct Kv8EvictParams {
  VbKv8Cache c;
  float *weights;
  int32_t *positions;
  const int32_t *lens;
  int32_t *lens_out;
  int32_t *status;
  int32_t *lists;            // per (sequence, head): holes, moving rows, first hole of a page
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
// All threads of the cluster meet; what they wrote, shared or global, is visible.
__device__ __forceinline__ void ev_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}
// A word of CTA `rank`'s shared memory.
__device__ __forceinline__ uint32_t ev_peer(const void *p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
  return r;
}

__global__ void __launch_bounds__(EV_THREADS) kv8_evict_kernel(const __grid_constant__ Kv8EvictParams p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_hist[2][EV_BINS];
  __shared__ uint32_t s_warp[2][EV_WARPS], s_total[3];  // total: ties; holes, moving rows
  __shared__ uint32_t s_bin, s_above, s_count;
  __shared__ int s_newest;
  __shared__ float s_edge[2];
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

  // ---- the newest position
  long long late = 0x7fffffffffffll;  // positions above it are protected
  if (p.recent > 0) {
    int newest = n - 1;
    if (positions) {
      newest = -0x7fffffff - 1;
      for (int t = 0; t < turns; ++t)
        if (row0 + t * 32 < n) newest = max(newest, positions[row0 + t * 32]);
      newest = __reduce_max_sync(0xffffffffu, newest);
      if (lane == 0) s_warp[0][warp] = (uint32_t)newest;
      __syncthreads();
      if (warp == 0) {
        newest = __reduce_max_sync(0xffffffffu, (int)s_warp[0][lane]);
        if (lane == 0) s_newest = newest;
      }
      ev_sync();
      for (uint32_t r = 0; r < C; ++r) newest = max(newest, (int)ev_peer(&s_newest, r));
    }
    late = (long long)newest - p.recent;
  }
  auto make_key = [&](int i) {
    const float w = weights[i] + 0.f;
    uint32_t k = __float_as_uint(w);
    k = w != w ? 0u : k >> 31 ? ~k : k | 0x80000000u;
    return i < p.first || (positions ? positions[i] : i) > late ? EV_SAFE : k;
  };
  auto key = [&](int t) {
    return at0 + t * 32 < p.cached ? s_keys[at0 + t * 32] : make_key(row0 + t * 32);
  };

  // ---- the key of the last row that stays: `need` of the rows that have it do
  uint32_t prefix = 0, need = (uint32_t)p.keep;
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {
    const int low = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
    uint32_t *hist = s_hist[d & 1];
    for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int t = 0; t < turns; ++t) {
      const int i = row0 + t * 32;
      if (i >= n) break;
      uint32_t k;
      if (d == 0) {
        k = make_key(i);
        if (at0 + t * 32 < p.cached) s_keys[at0 + t * 32] = k;
      } else {
        k = key(t);
      }
      if (d == 0 || k >> (low + bits) == prefix)
        atomicAdd(hist + ((k >> low) & ((1u << bits) - 1)), 1u);
    }
    ev_sync();
    // bins from the top: thread tid has 2047 - 2 tid and 2046 - 2 tid
    uint32_t hi = 0, lo = 0;
    for (uint32_t r = 0; r < C; ++r) {
      hi += ev_peer(hist + EV_BINS - 1 - 2 * tid, r);
      lo += ev_peer(hist + EV_BINS - 2 - 2 * tid, r);
    }
    uint32_t inc = hi + lo;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_warp[0][warp] = inc;
    __syncthreads();
    uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[0][lane] : 0u);
    before += inc - hi - lo;
    if (before < need && need <= before + hi + lo) {
      const bool upper = need <= before + hi;
      s_bin = EV_BINS - 1 - 2 * tid - (upper ? 0 : 1);
      s_above = before + (upper ? 0 : hi);
      s_count = upper ? hi : lo;
    }
    __syncthreads();
    need -= s_above;
    prefix = prefix << bits | s_bin;
    __syncthreads();  // s_warp, s_bin are free again
  }
  const uint32_t last = prefix;
  const bool ties = need < s_count;  // not all rows with the last key stay: the lower ones

  // Exclusive sums over the warps and CTAs before this warp of up to two counts.
  auto before = [&](uint32_t a, uint32_t c, int slot, uint32_t &sa, uint32_t &sc) {
    if (lane == 0) {
      s_warp[0][warp] = a;
      s_warp[1][warp] = c;
    }
    __syncthreads();
    const uint32_t ta = s_warp[0][lane], tc = s_warp[1][lane];
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
    ev_sync();
    for (uint32_t r = 0; r < rank; ++r) {
      sa += ev_peer(s_total + slot, r);
      if (slot) sc += ev_peer(s_total + 2, r);
    }
  };
  uint32_t tie0 = 0, unused;
  if (ties) {
    uint32_t mine = 0;
    for (int t = 0; t < turns; ++t)
      mine += __popc(__ballot_sync(0xffffffffu, row0 + t * 32 < n && key(t) == last));
    before(mine, 0, 0, tie0, unused);
  }
  const uint32_t below = (1u << lane) - 1;
  // whether row t of this lane stays; `tie`: rows with the last key before this turn
  auto stays = [&](int t, uint32_t &tie) {
    const bool there = row0 + t * 32 < n;
    const uint32_t k = there ? key(t) : 0u;
    if (!ties) return there && k >= last;
    const uint32_t same = __ballot_sync(0xffffffffu, there && k == last);
    const bool s = there && (k > last || (k == last && tie + __popc(same & below) < need));
    tie += __popc(same);
    return s;
  };
  uint32_t n_holes = 0, n_moving = 0, tie = tie0;
  for (int t = 0; t < turns; ++t) {
    const int i = row0 + t * 32;
    const bool s = stays(t, tie);
    n_holes += __popc(__ballot_sync(0xffffffffu, !s && i < p.keep));
    n_moving += __popc(__ballot_sync(0xffffffffu, s && i >= p.keep));
  }
  uint32_t hole, move;
  before(n_holes, n_moving, 1, hole, move);
  tie = tie0;
  for (int t = 0; t < turns; ++t) {
    const int i = row0 + t * 32;
    const bool s = stays(t, tie);
    const uint32_t hb = __ballot_sync(0xffffffffu, !s && i < p.keep);
    const uint32_t mb = __ballot_sync(0xffffffffu, s && i >= p.keep);
    if (i < p.keep && (i & (p.c.page - 1)) == 0)
      firsts[i >> p.shift] = (int)(hole + __popc(hb & below));
    if (i == p.keep - 1)  // the number of holes behind the last page
      firsts[(p.keep + p.c.page - 1) >> p.shift] = (int)(hole + __popc(hb & (below * 2 + 1)));
    if ((hb >> lane) & 1) holes[hole + __popc(hb & below)] = i;
    if ((mb >> lane) & 1) moving[move + __popc(mb & below)] = i;
    hole += __popc(hb);
    move += __popc(mb);
  }
  // the page in which `keep` falls: rows of it may move, and its scale may change
  const int edge = p.keep >> p.shift;
  if (tid < 2) {
    const int id = kv8_page(table, p.c.max_pages, p.c.pages, edge, nullptr);
    s_edge[tid] = id < 0 ? 0.f
                         : (tid ? p.c.v_scales : p.c.k_scales)[(size_t)id * p.c.kv_heads + h];
  }
  ev_sync();

  // ---- a warp takes a page of K or V at a time
  const int pages = (p.keep + p.c.page - 1) >> p.shift, D = p.c.dim, lpr = D >> 4;
  const size_t page_bytes = (size_t)p.c.page * D;
  for (int task = (int)rank * EV_WARPS + warp; task < 2 * pages; task += (int)C * EV_WARPS) {
    const int pg = task >> 1, kv = task & 1;
    const int j0 = __ldcg(firsts + pg), j1 = __ldcg(firsts + pg + 1);
    if (j0 == j1) continue;
    const int id = kv8_page(table, p.c.max_pages, p.c.pages, pg, lane == 0 ? p.status : nullptr);
    if (id < 0) continue;
    int8_t *codes = kv ? p.c.v_codes : p.c.k_codes;
    float *scales = kv ? p.c.v_scales : p.c.k_scales;
    int8_t *dst = codes + ((size_t)id * p.c.kv_heads + h) * page_bytes;
    const int live = min(p.c.page, p.keep - (pg << p.shift));
    const bool stay = j1 - j0 < live;
    const float old = pg == edge ? s_edge[kv] : scales[(size_t)id * p.c.kv_heads + h];
    float top = stay ? old : 0.f;
    // where the row of hole j comes from: its page and that page's scale
    auto from = [&](int j, int &src, int &sid, float &s) {
      src = __ldcg(moving + j);
      sid = kv8_page(table, p.c.max_pages, p.c.pages, src >> p.shift, p.status);
      s = sid < 0 ? 0.f : (src >> p.shift) == edge ? s_edge[kv]
                        : scales[(size_t)sid * p.c.kv_heads + h];
    };
    uint32_t filled[4] = {0, 0, 0, 0};  // rows of the page that are holes
    for (int j = j0; j < j1; j += 32) {
      uint32_t bit = 0;
      int word = 4;
      if (j + lane < j1) {
        int src, sid;
        float s;
        from(j + lane, src, sid, s);
        top = fmaxf(top, s);
        const int r = __ldcg(holes + j + lane) & (p.c.page - 1);
        word = r >> 5;
        bit = 1u << (r & 31);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
        filled[w] |= __reduce_or_sync(0xffffffffu, word == w ? bit : 0u);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (stay && top > old) {  // the rows that stay take the larger scale
      const float ratio = __fdiv_rn(old, top);
#pragma unroll 4
      for (int x = lane; x < live * lpr; x += 32) {
        const int r = x / lpr;
        const uint32_t f = r < 64 ? (r < 32 ? filled[0] : filled[1])
                                  : (r < 96 ? filled[2] : filled[3]);
        if ((f >> (r & 31)) & 1) continue;
        uint4 *at = reinterpret_cast<uint4 *>(dst) + x;
        *at = kv8_recode(*at, ratio);
      }
    }
    const int per = 32 / lpr, sub = lane / lpr, ch = lane % lpr;
    for (int j = j0; j < j1; j += 32) {
      int src = 0, sid = -1, row = 0;
      float s = 0.f;
      if (j + lane < j1) {
        from(j + lane, src, sid, s);
        row = __ldcg(holes + j + lane);
        if (kv == 0) {
          weights[row] = weights[src];
          if (positions) positions[row] = positions[src];
        }
      }
      const float ratio = top > 0.f ? __fdiv_rn(s, top) : 1.f;
      const int count = min(32, j1 - j);
#pragma unroll 4
      for (int k = 0; k < count; k += per) {
        const int o = k + sub;
        const int osrc = __shfl_sync(0xffffffffu, src, o & 31);
        const int osid = __shfl_sync(0xffffffffu, sid, o & 31);
        const int orow = __shfl_sync(0xffffffffu, row, o & 31);
        const float orat = __shfl_sync(0xffffffffu, ratio, o & 31);
        if (o >= count || osid < 0) continue;
        const uint4 x = *(reinterpret_cast<const uint4 *>(
                              codes + ((size_t)osid * p.c.kv_heads + h) * page_bytes +
                              (size_t)(osrc & (p.c.page - 1)) * D) + ch);
        *(reinterpret_cast<uint4 *>(dst + (size_t)(orow & (p.c.page - 1)) * D) + ch) =
            orat == 1.f ? x : kv8_recode(x, orat);
      }
    }
    if (lane == 0 && top != old) scales[(size_t)id * p.c.kv_heads + h] = top;
  }
}

struct EvictPlan {
  int cap, most, ctas, cached;
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
  pl.ctas = 1;
  while (pl.ctas < 8 && units * pl.ctas * 2 <= 148 && pl.cap > 2 * EV_THREADS * pl.ctas)
    pl.ctas *= 2;
  const long long per = align_up((pl.cap + pl.ctas - 1) / pl.ctas, EV_THREADS);
  pl.cached = (int)(per < EV_KEYS ? per : EV_KEYS);
  pl.stride = 2ll * pl.most + (a->keep + a->cache.page - 1) / a->cache.page + 1;
  pl.bytes = pl.most ? (size_t)(units * pl.stride) * sizeof(int32_t) : 0;
  return pl;
}

int ev_check(const VbKv8EvictArgs *a) {
  VB_REQUIRE(a, "vb_kv8_evict: null args");
  const int rc = kv8_check(&a->cache, "vb_kv8_evict");
  if (rc != VB_OK) return rc;
  VB_REQUIRE(a->keep >= 1 && a->room >= 0 && a->room <= 0x7fffffff - 65536,
             "vb_kv8_evict: keep=%d room=%d", a->keep, a->room);
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
  VB_REQUIRE(units * pl.ctas <= 0x7fffffffll, "vb_kv8_evict: too many sequences and heads");
  Kv8EvictParams p;
  p.c = a->cache;
  p.weights = a->weights; p.positions = a->positions;
  p.lens = a->lens; p.lens_out = a->lens_out; p.status = a->status;
  p.lists = static_cast<int32_t *>(a->workspace);
  p.list_stride = pl.stride; p.most = pl.most;
  p.room = a->room; p.cap = pl.cap; p.keep = a->keep; p.first = a->first; p.recent = a->recent;
  p.shift = kv8_page_shift(a->cache.page);
  p.cached = pl.cached;
  static std::atomic<uint64_t> ready{0};
  const int set = once_per_device(ready, [] {
    const cudaError_t e = cudaFuncSetAttribute(
        kv8_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_KEYS * 4);
    return e == cudaSuccess ? VB_OK
                            : set_error(VB_ERR_CUDA, "kv8_evict_kernel attributes: %s",
                                        cudaGetErrorString(e));
  });
  if (set != VB_OK) return set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * pl.ctas));
  cfg.blockDim = dim3(EV_THREADS);
  cfg.dynamicSmemBytes = (size_t)pl.cached * 4;
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pl.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kv8_evict_kernel, p);
  return check_launch("kv8_evict_kernel");
}

}  // extern "C"
