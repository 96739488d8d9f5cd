// Log probabilities of given tokens, their rank, the entropy and the best
// alternatives of every row, in one pass over the logits.
//
// With m the largest logit so far, c = log2(e) / T and y_j = (x_j - m) c:
//   s = sum 2^y_j,  t = sum 2^y_j y_j   (float32)
//   logprob = (x_t - m) / T - log2 s ln 2,  entropy = (log2 s - t / s) ln 2.
// When m moves, with d = (m_old - m_new) c: t <- 2^d (t + d s), s <- 2^d s, so
// the running maximum is carried per thread and the row is read once. Logits
// enter the sums at no less than -1e32 (2^y = 0 beside any larger one), which
// keeps 0 * inf out of t; NaN and +inf go through and give NaN. The difference
// is taken before the product: it is exactly 0 at the maximum however large the
// logits are. Instruction-bound before it is HBM-bound, so bf16 pairs are
// compared and clamped two at a time and the sums run on pairs of float32.
//
// Best alternatives: the k-th largest of the threads' own maxima is a lower
// bound v of the k-th largest logit (k threads hold one at least that large),
// so only threads whose maximum reaches v can hold any of the k best. Their
// vectors, about k / 256 of the row, are looked at again (they are in L2) and
// the logits >= v collected as 64-bit keys (ordered value, ~id), which have no
// ties; the k largest keys are the answer.
//
// One CTA per row, or per slice of a row when there are few rows: the last
// slice of a row (ticket) joins the slices in a fixed order.
//
// 2,048 rows of 151,936 bf16, top 20, take 153 to 168 us (3.7 to 4.1 TB/s, a copy 97):
// 12 instructions a logit, issue 66 %, exponentials 51 % of their pipe; float32 287 us
// (4.3 TB/s). 4 rows, top 5: 9.6 us on the device (float32 10.0), one row, top 32: 10.2.
#include "common.cuh"

namespace vb {
namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNROLL = 4;
constexpr int LP_MAX_TOP = 32;
constexpr int LP_SHORT = 8 * LP_THREADS;         // rows up to here go logit by logit
constexpr int LP_BATCH = LP_THREADS * 8;         // most keys one look can add
constexpr int LP_CAP = LP_BATCH + LP_MAX_TOP;
// Up to here every key is ranked at once, beyond it the k-th is bisected for first (one
// row, 304 keys: 16.6 us and 30.9; 30 rows, 608 keys: 38.3 and 36.2).
constexpr int LP_RANK_ALL = 512;
constexpr int LP_MAX_PARTS = 64;
constexpr int LP_CTAS = 4;                       // per SM: one's tail behind the others' loads
constexpr int LP_FILL = LP_CTAS * 148;
// bytes: a word per row of a split call
constexpr size_t LP_TICKETS = VB_TOKEN_LOGPROBS_WORKSPACE_HEAD;
static_assert(LP_FILL / 2 * sizeof(uint32_t) <= LP_TICKETS, "rows of a split call");
static_assert(LP_SHORT <= LP_CAP, "keys of a short row");
static_assert(LP_MAX_PARTS * LP_MAX_TOP <= LP_CAP, "keys of a split row");
// Least logit of the sums, and m at first: about -1e32, a bf16 value (0xF49E).
constexpr float LP_FLOOR = -1.0014439741803012e32f;
constexpr float LP_LN2 = 0.693147180559945309f;

struct LpStats {
  float m, s, t;  // maximum, sum, weighted sum
  float best;     // largest logit (NaN ignored), -inf if there is none above it
  int32_t ahead;  // logits ahead of the token
  int32_t pad[3];
};

struct LpParams {
  const void *logits;
  const int32_t *tokens;
  float *logprob, *entropy, *top_logprobs;
  int32_t *rank, *top_ids, *status;
  LpStats *part_stats;            // [rows, parts]
  unsigned long long *part_keys;  // [rows, parts, top]
  uint32_t *tickets;              // [rows], zero between calls
  int64_t row_stride;
  float c, inv_t;                 // log2(e) / temperature, 1 / temperature
  int vocab, top, parts;
};

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Unsigned order of floats (NaN as -inf, -0 as 0).
__device__ __forceinline__ uint32_t lp_order(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_unorder(uint32_t o) {
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ unsigned long long lp_key(float x, int id) {
  return ((unsigned long long)lp_order(x) << 32) | (uint32_t)~id;
}
// The next larger value of the type (NaN after +inf and NaN: nothing compares).
__device__ __forceinline__ float lp_next(float x, bool bf16) {
  if (x != x) return x;
  const uint32_t step = bf16 ? 0x10000u : 1u;
  if (x == 0.f) return __uint_as_float(step);
  const uint32_t u = __float_as_uint(x);
  if (u == 0x7F800000u) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((u & 0x80000000u) ? u - step : u + step);
}

// 16 bytes of a row: 8 bf16 or 4 float32 values. `bar` is what a logit has to
// reach to count as ahead of the token, in the form of the type.
template <typename T>
struct LpVec;
template <>
struct LpVec<uint16_t> {
  static constexpr int N = 8;
  static constexpr bool BF16 = true;
  static constexpr uint32_t NONE = 0xFF80FF80u;  // -inf
  static constexpr uint32_t NO_BAR = 0x7FC07FC0u;
  __device__ static uint32_t bar(float x) { return (__float_as_uint(x) >> 16) * 0x10001u; }
  __device__ static float at(const uint4 &v, int j) {
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    return __uint_as_float((j & 1) ? (w & 0xFFFF0000u) : (w << 16));
  }
  __device__ static float load(const uint16_t *p) { return bf2f(*p); }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {  // NaN loses
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  // largest of a vector's logits and r
  __device__ static void top(uint32_t &r, const uint4 &v) {
    r = max2(r, max2(max2(v.x, v.y), max2(v.z, v.w)));
  }
  __device__ static float top_value(uint32_t r) {
    return fmaxf(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
  }
  // the j-th pair of a vector, no less than LP_FLOOR (NaN stays)
  static constexpr int PAIRS = 4;
  __device__ static f2 pair(const uint4 &v, int j) {
    uint32_t w = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0xF49EF49Eu));  // LP_FLOOR
    return f2_make(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  // number of a vector's logits that reach the bar, added to two bf16 counts
  // (exact up to 256 each)
  __device__ static void count(uint32_t &n, const uint4 &v, uint32_t bar) {
    uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      asm("set.ge.bf16x2.bf16x2 %0, %0, %1;" : "+r"(x[j]) : "r"(bar));
      asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(n) : "r"(x[j]));
    }
  }
  __device__ static int counted(uint32_t n) {
    return (int)(__uint_as_float(n << 16) + __uint_as_float(n & 0xFFFF0000u));
  }
};
template <>
struct LpVec<float> {
  static constexpr int N = 4;
  static constexpr bool BF16 = false;
  static constexpr uint32_t NONE = 0xFF800000u;
  static constexpr uint32_t NO_BAR = 0x7FC00000u;
  __device__ static uint32_t bar(float x) { return __float_as_uint(x); }
  __device__ static float at(const uint4 &v, int j) {
    return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
  __device__ static float load(const float *p) { return *p; }
  __device__ static void top(uint32_t &r, const uint4 &v) {
    r = __float_as_uint(fmaxf(fmaxf(fmaxf(__uint_as_float(r), at(v, 0)), at(v, 1)),
                              fmaxf(at(v, 2), at(v, 3))));
  }
  __device__ static float top_value(uint32_t r) { return __uint_as_float(r); }
  static constexpr int PAIRS = 2;
  __device__ static f2 pair(const uint4 &v, int j) {
    float a = at(v, 2 * j), b = at(v, 2 * j + 1);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(LP_FLOOR));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(LP_FLOOR));
    return f2_make(a, b);
  }
  __device__ static void count(uint32_t &n, const uint4 &v, uint32_t bar) {
#pragma unroll
    for (int j = 0; j < 4; ++j) n += at(v, j) >= __uint_as_float(bar);
  }
  __device__ static int counted(uint32_t n) { return (int)n; }
};

// A row's vectors: vector v holds ids [v N - off, v N - off + N); those outside
// [0, vocab) are not part of the row (first and last vector only).
template <typename T>
struct LpRow {
  const T *x;
  int off, nvec, w_lo, w_hi;  // whole vectors: [w_lo, w_hi)
  __device__ LpRow(const void *logits, int64_t row, int64_t stride, int n) {
    x = static_cast<const T *>(logits) + row * stride;
    off = (int)(((uintptr_t)x & 15) / sizeof(T));
    nvec = (n + off + LpVec<T>::N - 1) / LpVec<T>::N;
    w_lo = off > 0;
    w_hi = (n + off) / LpVec<T>::N;
  }
  // where vector v begins: inside the row for whole vectors, which alone are read
  __device__ const uint4 *at(int v) const {
    return reinterpret_cast<const uint4 *>(reinterpret_cast<uintptr_t>(x) & ~uintptr_t(15)) + v;
  }
};

__device__ __forceinline__ void lp_move(float &m, float &s, float &t, float to, float c) {
  if (to > m) {
    const float d = fmaxf((m - to) * c, -1000.f), a = lp_ex2(d);
    t = a * fmaf(d, s, t);
    s = a * s;
    m = to;
  }
}
__device__ __forceinline__ void lp_join(float &m, float &s, float &t, float m2, float s2,
                                        float t2, float c) {
  const float to = fmaxf(m, m2);
  lp_move(m, s, t, to, c);
  lp_move(m2, s2, t2, to, c);
  s += s2;
  t += t2;
}

// The k largest of buf[0, n) (distinct keys) in descending order into list;
// zeros beyond n. Called by every thread; buf and list are reusable after the
// closing barrier.
__device__ void lp_select(unsigned long long *buf, int n, int k, unsigned long long *list,
                          unsigned long long *tmp, int *s_n, int *s_cnt) {
  const int tid = threadIdx.x;
  if (n > LP_RANK_ALL) {  // many candidates (ties): bisect for the k-th key first
    unsigned long long thr = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const unsigned long long cand = thr | (1ull << bit);
      int c = 0;
      for (int i = tid; i < n; i += LP_THREADS) c += buf[i] >= cand;
      c = __reduce_add_sync(0xffffffffu, c);
      if ((tid & 31) == 0) s_cnt[tid >> 5] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < LP_WARPS; ++w) c += s_cnt[w];
      if (c >= k) thr = cand;
      __syncthreads();
    }
    if (tid == 0) *s_n = 0;
    __syncthreads();
    for (int i = tid; i < n; i += LP_THREADS)
      if (buf[i] >= thr) tmp[atomicAdd(s_n, 1)] = buf[i];  // exactly k
    __syncthreads();
    if (tid < k) buf[tid] = tmp[tid];
    n = k;
    __syncthreads();
  }
  if (tid >= n && tid < k) list[tid] = 0;
  for (int i = tid; i < n; i += LP_THREADS) {
    const unsigned long long key = buf[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += buf[j] > key;
    if (r < k) list[r] = key;
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) token_logprobs_kernel(LpParams p) {
  using V = LpVec<T>;
  __shared__ unsigned long long s_buf[LP_CAP];
  __shared__ unsigned long long s_list[LP_MAX_TOP], s_tmp[LP_MAX_TOP];
  __shared__ float s_m[LP_WARPS], s_s[LP_WARPS], s_t[LP_WARPS], s_b[LP_WARPS];
  __shared__ int s_a[LP_WARPS], s_cnt[LP_WARPS];
  __shared__ uint16_t s_owner[LP_THREADS];
  __shared__ int s_n, s_owners, s_last;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const LpRow<T> r(p.logits, row, p.row_stride, p.vocab);
  const int v_lo = (int)((int64_t)r.nvec * part / p.parts);
  const int v_hi = (int)((int64_t)r.nvec * (part + 1) / p.parts);
  // whole vectors [w_lo, w_hi), thread t takes w_lo + t + i LP_THREADS; the
  // row's ragged ends, if this slice has them, are looked at logit by logit
  // (a short row all of it, thread t the ids t + i LP_THREADS)
  const bool brief = p.vocab <= LP_SHORT;
  const int w_lo = max(v_lo, r.w_lo), w_hi = brief ? w_lo : max(w_lo, min(v_hi, r.w_hi));
  const int end0 = !brief && v_lo < r.w_lo ? 0 : -1;
  const int end1 = !brief && v_hi == r.nvec && r.w_hi < r.nvec ? r.w_hi : -1;
  constexpr int STEP = LP_THREADS * LP_UNROLL;
  const int n_full = (w_hi - w_lo) / STEP;  // turns in which every thread has LP_UNROLL vectors
  const float c = p.c;

  const int tok = p.tokens[row];
  const uint4 *src = r.at(w_lo + tid);
  uint4 next[LP_UNROLL];
  auto fetch = [&](int turn) {
    if (turn < n_full) {
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) next[u] = ldg_nc_v4(src + u * LP_THREADS);
    } else {  // the last turn, short of vectors
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) {
        next[u] = make_uint4(V::NONE, V::NONE, V::NONE, V::NONE);
        if (w_lo + turn * STEP + u * LP_THREADS + tid < w_hi)
          next[u] = ldg_nc_v4(src + u * LP_THREADS);
      }
    }
    src += STEP;
  };
  fetch(0);
  const bool tok_ok = (unsigned)tok < (unsigned)p.vocab;
  const float xt = tok_ok ? V::load(r.x + tok) : 0.f;
  const float xt_next = lp_next(xt, V::BF16);
  const int tok_vec = tok_ok ? (tok + r.off) / V::N : -1;
  // ids below the token's count when equal; without a token (or a NaN) nothing does
  const uint32_t bar_lo = tok_ok ? V::bar(xt) : V::NO_BAR;
  const uint32_t bar_hi = tok_ok ? V::bar(xt_next) : V::NO_BAR;

  float m = LP_FLOOR, s = 0.f, t = 0.f, best = -INFINITY;
  int ahead = 0;
  {
    const f2 cc = f2_make(c, c);
    f2 ss = 0, tt = 0;
    const int turns = n_full + (n_full * STEP < w_hi - w_lo);
    for (int turn = 0; turn < turns; ++turn) {
      uint4 x[LP_UNROLL];
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) x[u] = next[u];
      if (turn + 1 < turns) fetch(turn + 1);
      uint32_t top = V::NONE;
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u) V::top(top, x[u]);
      const float top_x = V::top_value(top);
      best = fmaxf(best, top_x);
      if (top_x > m) {
        float s0, s1, t0, t1;
        f2_split(ss, s0, s1);
        f2_split(tt, t0, t1);
        s = s0 + s1;
        t = t0 + t1;
        lp_move(m, s, t, top_x, c);
        ss = f2_make(s, 0.f);
        tt = f2_make(t, 0.f);
      }
      if (top_x >= xt) {  // some logit may be ahead of the token
        uint32_t n = 0;
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
          const int v = w_lo + turn * STEP + u * LP_THREADS + tid;
          V::count(n, x[u], v >= w_hi ? V::NO_BAR : v < tok_vec ? bar_lo : bar_hi);
        }
        ahead += V::counted(n);
      }
      const f2 mm = f2_make(-m, -m);
#pragma unroll
      for (int u = 0; u < LP_UNROLL; ++u)
#pragma unroll
        for (int j = 0; j < V::PAIRS; ++j) {
          const f2 y = f2_mul(f2_add(V::pair(x[u], j), mm), cc);
          float y0, y1;
          f2_split(y, y0, y1);
          const f2 e = f2_make(lp_ex2(y0), lp_ex2(y1));
          ss = f2_add(ss, e);
          tt = f2_fma(e, y, tt);
        }
    }
    float s0, s1, t0, t1;
    f2_split(ss, s0, s1);
    f2_split(tt, t0, t1);
    s = s0 + s1;
    t = t0 + t1;
    auto one = [&](int id, bool first) {  // first: ahead when equal
      const float f = V::load(r.x + id);
      best = fmaxf(best, f);
      lp_move(m, s, t, f, c);
      const float y = ((f < LP_FLOOR ? LP_FLOOR : f) - m) * c, e = lp_ex2(y);
      s += e;
      t = fmaf(e, y, t);
      ahead += tok_ok && (first ? f >= xt : f >= xt_next);
    };
    if (brief)
      for (int id = tid; id < p.vocab; id += LP_THREADS) one(id, id < tok);
    auto ragged = [&](int v) {
      for (int j = 0; j < V::N; ++j) {
        const int id = v * V::N - r.off + j;
        if (id >= 0 && id < p.vocab) one(id, v < tok_vec);
      }
    };
    if (end0 >= 0 && tid == 0) ragged(end0);
    if (end1 >= 0 && tid == 1) ragged(end1);
    // equal logits of lower id in the token's own vector
    if (!brief && tok_ok && tid == 2 && tok_vec >= v_lo && tok_vec < v_hi)
      for (int id = max(0, tok_vec * V::N - r.off); id < tok; ++id)
        ahead += V::load(r.x + id) == xt;
  }

  // ---- the k best of this slice
  const int k = p.top;
  if (k > 0) {
    const uint32_t mine = lp_order(best);  // (-inf for a thread without vectors)
    uint32_t thr = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t cand = thr | (1u << bit);
      if (__syncthreads_count(mine >= cand) >= k) thr = cand;
    }
    if (tid == 0) s_owners = s_n = 0;
    __syncthreads();
    if (mine >= thr && w_lo + tid < w_hi) s_owner[atomicAdd(&s_owners, 1)] = (uint16_t)tid;
    __syncthreads();
    const int owners = s_owners;
    const int items = owners * ((w_hi - w_lo + LP_THREADS - 1) / LP_THREADS) + 2;
    auto keep = [&](float f, int id, unsigned long long least) {
      if (lp_order(f) < thr) return;
      const unsigned long long key = lp_key(f, id);
      if (key <= least) return;
      const int at = atomicAdd(&s_n, 1);
      if (at < LP_CAP) s_buf[at] = key;
    };
    // keys of item i that reach the bounds: vector (i - 2) / owners of an owner,
    // items 0 and 1 the ragged ends
    auto look = [&](int i, unsigned long long least) {
      int v;
      if (i < 2) {
        v = i ? end1 : end0;
        if (v < 0) return;
      } else {
        v = w_lo + (i - 2) / owners * LP_THREADS + s_owner[(i - 2) % owners];
        if (v >= w_hi) return;
      }
      uint4 x = make_uint4(0, 0, 0, 0);
      if (i >= 2) x = ldg_nc_v4(r.at(v));
#pragma unroll
      for (int j = 0; j < V::N; ++j) {
        const int id = v * V::N - r.off + j;
        if (id < 0 || id >= p.vocab) continue;
        keep(i >= 2 ? V::at(x, j) : V::load(r.x + id), id, least);
      }
    };
    if (brief)  // (at most LP_SHORT keys)
      for (int id = tid; id < p.vocab; id += LP_THREADS) keep(V::load(r.x + id), id, 0);
    else
#pragma unroll 2
    for (int i = tid; i < items; i += LP_THREADS) look(i, 0);
    __syncthreads();
    int n = s_n;
    if (n <= LP_CAP) {
      lp_select(s_buf, n, k, s_list, s_tmp, &s_n, s_cnt);
    } else {  // (many equal logits) look again, a bounded number of keys at a time
      __syncthreads();
      if (tid == 0) s_n = 0;
      __syncthreads();
      unsigned long long kth = 0;
      for (int i0 = 0; i0 < items; i0 += LP_THREADS) {
        if (i0 + tid < items) look(i0 + tid, kth);
        __syncthreads();
        n = s_n;
        const bool last = i0 + LP_THREADS >= items;
        if (last || n > LP_CAP - LP_BATCH) {
          lp_select(s_buf, n, k, s_list, s_tmp, &s_n, s_cnt);
          const int have = min(n, k);
          if (have == k) kth = s_list[k - 1];
          if (!last) {
            if (tid < have) s_buf[tid] = s_list[tid];
            if (tid == 0) s_n = have;
          }
        }
        __syncthreads();
      }
    }
  }

  // ---- sums over the CTA
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o),
                t2 = __shfl_xor_sync(0xffffffffu, t, o);
    lp_join(m, s, t, m2, s2, t2, c);
    best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  }
  ahead = __reduce_add_sync(0xffffffffu, ahead);
  if ((tid & 31) == 0) {
    s_m[tid >> 5] = m; s_s[tid >> 5] = s; s_t[tid >> 5] = t;
    s_b[tid >> 5] = best; s_a[tid >> 5] = ahead;
  }
  __syncthreads();
  if (tid < 32) {  // lane w < 16 holds warp w's, the others nothing
    const int w = tid & (LP_WARPS - 1);
    m = s_m[w]; s = tid < LP_WARPS ? s_s[w] : 0.f; t = tid < LP_WARPS ? s_t[w] : 0.f;
    best = s_b[w];
    ahead = tid < LP_WARPS ? s_a[w] : 0;
#pragma unroll
    for (int o = LP_WARPS / 2; o > 0; o >>= 1) {
      const float m2 = __shfl_down_sync(0xffffffffu, m, o);
      const float s2 = __shfl_down_sync(0xffffffffu, s, o);
      const float t2 = __shfl_down_sync(0xffffffffu, t, o);
      lp_join(m, s, t, m2, s2, t2, c);
      best = fmaxf(best, __shfl_down_sync(0xffffffffu, best, o));
      ahead += __shfl_down_sync(0xffffffffu, ahead, o);
    }
  }
  if (p.parts > 1) {  // leave the slice's sums and keys; the row's last slice joins them
    const size_t at = (size_t)row * p.parts + part;
    if (tid == 0) {
      LpStats st;
      st.m = m; st.s = s; st.t = t; st.best = best; st.ahead = ahead;
      st.pad[0] = st.pad[1] = st.pad[2] = 0;
      p.part_stats[at] = st;
    }
    if (tid < k) p.part_keys[at * k + tid] = s_list[tid];
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      s_last = atomicAdd(p.tickets + row, 1u) == (uint32_t)p.parts - 1;
      if (s_last) p.tickets[row] = 0;
      s_n = 0;
      s_tmp[0] = ~0ull;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    if (k > 0) {
      const unsigned long long *keys = p.part_keys + (size_t)row * p.parts * k;
      // The lists are in descending order: with j * parts >= k, at least k keys reach
      // the least of the slices' j-th ones, and only those are looked at (19 slices,
      // 20 best: some 80 of 380).
      if (tid < p.parts)
        atomicMin(s_tmp, __ldcg(keys + tid * k + (k + p.parts - 1) / p.parts - 1));
      __syncthreads();
      const unsigned long long least = s_tmp[0];
#pragma unroll 2
      for (int i = tid; i < p.parts * k; i += LP_THREADS) {
        const unsigned long long key = __ldcg(keys + i);
        if (key && key >= least) s_buf[atomicAdd(&s_n, 1)] = key;
      }
      __syncthreads();
      const int n = s_n;
      lp_select(s_buf, n, k, s_list, s_tmp, &s_n, s_cnt);
    }
    if (tid < 32) {  // lane i takes slices i and i + 32
      const LpStats *st = p.part_stats + (size_t)row * p.parts;
      m = LP_FLOOR; s = t = 0.f; best = -INFINITY; ahead = 0;
#pragma unroll
      for (int i = 0; i < LP_MAX_PARTS; i += 32) {
        if (i + tid >= p.parts) continue;
        const float4 a = __ldcg(reinterpret_cast<const float4 *>(st + i + tid));
        lp_join(m, s, t, a.x, a.y, a.z, c);
        best = fmaxf(best, a.w);
        ahead += __ldcg(&st[i + tid].ahead);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
        const float s2 = __shfl_xor_sync(0xffffffffu, s, o);
        const float t2 = __shfl_xor_sync(0xffffffffu, t, o);
        lp_join(m, s, t, m2, s2, t2, c);
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
      }
      ahead = __reduce_add_sync(0xffffffffu, ahead);
    }
  }
  if (tid == 0) {
    s_b[0] = best;
    s_m[0] = m;
    s_s[0] = s;
    s_t[0] = t;
  }
  __syncthreads();
  best = s_b[0]; m = s_m[0]; s = s_s[0]; t = s_t[0];
  // Every logit of the row counted as LP_FLOOR. There the least difference of two values
  // is beyond any exponent, so those equal to the largest one share the probability.
  if (best <= LP_FLOOR && best > -INFINITY) {
    int n = 0;
    for (int id = tid; id < p.vocab; id += LP_THREADS) n += V::load(r.x + id) == best;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0) s_cnt[tid >> 5] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) n += s_cnt[w];
    // (a NaN in the row has come to s)
    s = s == s ? (float)n : s;
    t = 0.f;
    m = best;
  }
  const float lse = best == -INFINITY ? NAN : log2f(s) * LP_LN2;  // of the logits less m
  if (tid == 0) {
    p.logprob[row] = tok_ok ? (xt - m) * p.inv_t - lse : NAN;
    p.entropy[row] = lse - t / s * LP_LN2;
    p.rank[row] = tok_ok ? ahead : -1;
    if (!tok_ok) flag_status(p.status, VB_STATUS_BOUNDS);
  }
  if (tid < k) {
    const unsigned long long key = s_list[tid];
    p.top_ids[(size_t)row * k + tid] = (int32_t)~(uint32_t)key;
    p.top_logprobs[(size_t)row * k + tid] =
        (lp_unorder((uint32_t)(key >> 32)) - m) * p.inv_t - lse;
  }
}

// Slices per row: one CTA per row once the rows alone fill the GPU, else
// slices of at least one turn of the loop (bf16 vectors).
int lp_parts(int rows, int vocab) {
  const int most = (vocab - 1) / (LP_THREADS * LP_UNROLL * 8) + 1;
  int parts = rows > 0 ? LP_FILL / rows : 1;
  if (parts > most) parts = most;
  return parts < 1 ? 1 : parts > LP_MAX_PARTS ? LP_MAX_PARTS : parts;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" {

size_t vb_token_logprobs_workspace_size(int32_t rows, int32_t vocab, int32_t top) {
  if (rows < 1 || vocab < 1 || top < 0 || top > LP_MAX_TOP) return 0;
  const size_t parts = lp_parts(rows, vocab);
  return LP_TICKETS +
         (parts > 1 ? rows * parts * (sizeof(LpStats) + top * sizeof(unsigned long long)) : 0);
}

int vb_token_logprobs(const VbTokenLogprobsArgs *a, vb_stream_t stream) {
  VB_REQUIRE(a, "vb_token_logprobs: null args");
  VB_REQUIRE(a->rows >= 0 && a->rows <= (1 << 24) && a->vocab >= 1 && a->vocab <= (1 << 30),
             "vb_token_logprobs: rows=%d (<= 2^24) vocab=%d (<= 2^30)", a->rows, a->vocab);
  VB_REQUIRE(a->top >= 0 && a->top <= LP_MAX_TOP && a->top <= a->vocab,
             "vb_token_logprobs: top=%d (at most %d and the vocabulary)", a->top, LP_MAX_TOP);
  VB_REQUIRE(a->dtype == 0 || a->dtype == 1, "vb_token_logprobs: dtype %d", a->dtype);
  VB_REQUIRE(a->temperature >= 1e-3f && a->temperature <= 1e3f,
             "vb_token_logprobs: temperature %g (1e-3 .. 1e3)", (double)a->temperature);
  if (a->rows == 0) return VB_OK;
  VB_REQUIRE(a->logits && a->tokens && a->logprob && a->entropy && a->rank &&
                 (a->top == 0 || (a->top_ids && a->top_logprobs)),
             "vb_token_logprobs: null tensor");
  VB_REQUIRE(((uintptr_t)a->logits % (a->dtype ? 4 : 2)) == 0,
             "vb_token_logprobs: logits not aligned to their type");
  VB_REQUIRE(a->row_stride >= a->vocab || a->rows == 1 || a->row_stride == 0,
             "vb_token_logprobs: row stride %lld below the vocabulary", (long long)a->row_stride);
  const size_t need = vb_token_logprobs_workspace_size(a->rows, a->vocab, a->top);
  if (!a->workspace || a->workspace_bytes < need)
    return set_error(VB_ERR_WORKSPACE, "vb_token_logprobs: workspace %zu < %zu bytes",
                     a->workspace_bytes, need);
  VB_REQUIRE(((uintptr_t)a->workspace % 16) == 0, "vb_token_logprobs: workspace alignment");
  LpParams p;
  p.logits = a->logits; p.tokens = a->tokens;
  p.logprob = a->logprob; p.entropy = a->entropy; p.top_logprobs = a->top_logprobs;
  p.rank = a->rank; p.top_ids = a->top_ids; p.status = a->status;
  p.parts = lp_parts(a->rows, a->vocab);
  uint8_t *w = static_cast<uint8_t *>(a->workspace);
  p.tickets = reinterpret_cast<uint32_t *>(w);
  w += LP_TICKETS;
  p.part_stats = reinterpret_cast<LpStats *>(w);
  w += (size_t)a->rows * p.parts * sizeof(LpStats);
  p.part_keys = reinterpret_cast<unsigned long long *>(w);
  p.row_stride = a->row_stride;
  p.c = (float)(1.4426950408889634 / (double)a->temperature);
  p.inv_t = (float)(1.0 / (double)a->temperature);
  p.vocab = a->vocab; p.top = a->top;
  const dim3 grid(a->rows * p.parts), block(LP_THREADS);
  if (a->dtype == 0)
    vb_launch(token_logprobs_kernel<uint16_t>, grid, block, 0, as_stream(stream), true, p);
  else
    vb_launch(token_logprobs_kernel<float>, grid, block, 0, as_stream(stream), true, p);
  return check_launch("token_logprobs_kernel");
}

}  // extern "C"
