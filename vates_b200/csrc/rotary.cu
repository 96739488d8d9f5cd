// Rotary positions with several axes for given tokens, after an optional RMS
// norm of every row (the input side of attention, for q and k in one launch).
//
//   y = x * rsqrt(mean(x^2) + eps) * w                 (y = x without a norm)
//   angle(t, i) = position[axis(i)][t] * base^(-2 i / R),   i < R / 2
//   (y_i, y_{i + R/2}) -> (y_i cos - y_{i+R/2} sin, y_{i+R/2} cos + y_i sin)
//
// Everything is float32 from the bf16 input to the one rounding at the end.
// The angle is taken in double and in turns: position * frequency is reduced to
// [-1/2, 1/2] before it becomes a float, so a token at position 10^7 (where a
// float32 product is off by whole radians) is as exact as one at 10.
#include "common.cuh"

namespace vb {
namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_PAIRS = 128;      // most rotated pairs of a row
constexpr int RT_TABLE = 2048;     // (token, pair) sines and cosines of a CTA
constexpr int RT_TOKENS = 32;      // most tokens of a CTA
constexpr int RT_AHEAD = 2;        // rows that a thread has in flight

struct RotateParams {
  const uint16_t *src[2];          // q, k
  uint16_t *dst[2];
  const uint16_t *norm[2];
  int64_t s_in[2][3], s_out[2][3]; // element strides of batch, head, row
  const int32_t *positions;        // [axes][tokens]
  int64_t tokens;                  // batch * L
  int L, heads[2], dim, half, per, groups;  // tokens of a CTA, CTAs of a sequence
  float eps;
  bool keep;                       // dims from R on are in place already
  double turns[RT_PAIRS];          // frequency / 2 pi
  uint8_t axis[RT_PAIRS];
};

// 8 bf16
__device__ __forceinline__ uint4 rt_load(const uint16_t *p, bool vec) {
  if (vec) return ldg_v4(p);
  return make_uint4(p[0] | ((uint32_t)p[1] << 16), p[2] | ((uint32_t)p[3] << 16),
                    p[4] | ((uint32_t)p[5] << 16), p[6] | ((uint32_t)p[7] << 16));
}
__device__ __forceinline__ void rt_floats(float (&x)[8], const uint4 &v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(w[j] << 16);
    x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void rt_store(uint16_t *p, const float (&x)[8], bool vec) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = pack_bf2(x[2 * j], x[2 * j + 1]);
  if (vec) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[2 * j] = (uint16_t)w[j];
      p[2 * j + 1] = (uint16_t)(w[j] >> 16);
    }
  }
}

// LPR lanes hold a row, 16 dims each: the first R / 16 of them 8 pairs, the
// others 16 dims that only the norm changes. A CTA takes some tokens of one
// sequence, all heads: it makes their sines once, and then goes through the rows
// head by head, so that what it writes to [batch, heads, L, dim] is contiguous.
template <int LPR, bool NORM>
__global__ void __launch_bounds__(RT_THREADS, 4) rotate_kernel(const __grid_constant__ RotateParams p,
                                                            bool vec) {
  __shared__ float2 s_cs[RT_TABLE];  // [token][pair % 8][pair / 8]
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const int b = blockIdx.x / p.groups, i0 = (blockIdx.x - b * p.groups) * p.per;
  const int n = min(p.per, p.L - i0);
  const uint32_t n_inv = (uint32_t)(0xFFFFFFFFu / n) + 1;  // r / n for r * n < 2^32; n = 1: 0
  const int j = tid % LPR, turned = p.half >> 3;
  // dims of this lane: two runs of eight
  const int d0 = j < turned ? j * 8 : 2 * p.half + (j - turned) * 16;
  const int d1 = j < turned ? p.half + j * 8 : d0 + 8;
  const bool live = j * 16 < p.dim && !(p.keep && j >= turned);
  constexpr int STEP = RT_THREADS / LPR;
  const int rows = n * (p.heads[0] + p.heads[1]);
  // row r: token, q (0) or k (1), and head
  auto place = [&](int r, int &t, int &kind, int &h) {
    const int hh = n == 1 ? r : (int)__umulhi((uint32_t)r, n_inv);
    t = r - hh * n;
    kind = hh >= p.heads[0];
    h = kind ? hh - p.heads[0] : hh;
  };
  auto fetch = [&](int r0, uint4 (&x)[RT_AHEAD], uint4 (&y)[RT_AHEAD]) {
#pragma unroll
    for (int k = 0; k < RT_AHEAD; ++k) {
      const int r = r0 + k * STEP;
      x[k] = y[k] = make_uint4(0, 0, 0, 0);
      if (r < rows && live) {
        int t, kind, h;
        place(r, t, kind, h);
        const int64_t *st = p.s_in[kind];
        const uint16_t *src = p.src[kind] + b * st[0] + h * st[1] + (i0 + t) * st[2];
        x[k] = rt_load(src + d0, vec);
        y[k] = rt_load(src + d1, vec);
      }
    }
  };
  uint4 x[RT_AHEAD], y[RT_AHEAD];
  fetch(tid / LPR, x, y);
  // sines while the first rows are on their way
  for (int z = tid; z < n * p.half; z += RT_THREADS) {
    const int t = z / p.half, i = z - t * p.half;
    const double turn = p.positions[p.axis[i] * p.tokens + (int64_t)b * p.L + i0 + t] * p.turns[i];
    float2 cs;
    sincospif(2.f * (float)(turn - rint(turn)), &cs.y, &cs.x);
    s_cs[t * p.half + (i & 7) * turned + (i >> 3)] = cs;
  }
  __syncthreads();
  for (int r0 = tid / LPR; r0 - tid / LPR < rows; r0 += STEP * RT_AHEAD) {
#pragma unroll
    for (int k = 0; k < RT_AHEAD; ++k) {
      const int r = r0 + k * STEP;
      int t, kind, h;
      place(r, t, kind, h);
      float u[8], v[8];
      rt_floats(u, x[k]);
      rt_floats(v, y[k]);
      if constexpr (NORM) {
        const uint16_t *w = p.norm[kind];
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(u[e], u[e], fmaf(v[e], v[e], ss));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && live) {
          const float inv = rsqrtf(ss / p.dim + p.eps);
          float wu[8], wv[8];
          rt_floats(wu, rt_load(w + d0, vec));
          rt_floats(wv, rt_load(w + d1, vec));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u[e] *= inv * wu[e];
            v[e] *= inv * wv[e];
          }
        }
      }
      if (r >= rows || !live) continue;
      if (j < turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 cs = s_cs[t * p.half + e * turned + j];
          const float c = u[e], s = v[e];
          u[e] = fmaf(c, cs.x, -s * cs.y);
          v[e] = fmaf(s, cs.x, c * cs.y);
        }
      }
      const int64_t *st = p.s_out[kind];
      uint16_t *dst = p.dst[kind] + b * st[0] + h * st[1] + (i0 + t) * st[2];
      rt_store(dst + d0, u, vec);
      rt_store(dst + d1, v, vec);
    }
    if (r0 - tid / LPR + STEP * RT_AHEAD < rows) fetch(r0 + STEP * RT_AHEAD, x, y);
  }
}

template <int LPR>
void rt_launch(const RotateParams &p, unsigned ctas, bool vec, cudaStream_t s) {
  if (p.norm[0] || p.norm[1])
    vb_launch(rotate_kernel<LPR, true>, dim3(ctas), dim3(RT_THREADS), 0, s, true, p, vec);
  else
    vb_launch(rotate_kernel<LPR, false>, dim3(ctas), dim3(RT_THREADS), 0, s, true, p, vec);
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" int vb_rotate_axes(const VbRotateArgs *a, vb_stream_t stream) {
  VB_REQUIRE(a, "vb_rotate_axes: null args");
  VB_REQUIRE(a->dim >= 16 && a->dim <= 256 && a->dim % 16 == 0,
             "vb_rotate_axes: head dim %d (16 to 256, a multiple of 16)", a->dim);
  VB_REQUIRE(a->rope_dims >= 16 && a->rope_dims <= a->dim && a->rope_dims % 16 == 0,
             "vb_rotate_axes: %d rotated dims of %d (a multiple of 16)", a->rope_dims, a->dim);
  VB_REQUIRE(a->batch >= 0 && a->L >= 0 && a->q_heads >= 0 && a->kv_heads >= 0 &&
                 a->q_heads <= 32768 && a->kv_heads <= 32768,
             "vb_rotate_axes: batch=%d L=%d heads=%d, %d", a->batch, a->L, a->q_heads,
             a->kv_heads);
  VB_REQUIRE(a->axes >= 1 && a->axes <= 255, "vb_rotate_axes: %d axes (1 to 255)", a->axes);
  VB_REQUIRE(a->eps >= 0.f && a->eps < 1e30f, "vb_rotate_axes: eps %g", (double)a->eps);
  VB_REQUIRE(a->turns && a->axis, "vb_rotate_axes: null table");
  RotateParams p = {};
  p.half = a->rope_dims / 2;
  for (int i = 0; i < p.half; ++i) {
    VB_REQUIRE(a->axis[i] < a->axes, "vb_rotate_axes: pair %d on axis %d of %d", i, a->axis[i],
               a->axes);
    VB_REQUIRE(a->turns[i] > -1e6 && a->turns[i] < 1e6, "vb_rotate_axes: frequency %g of pair %d",
               a->turns[i], i);
    p.turns[i] = a->turns[i];
    p.axis[i] = a->axis[i];
  }
  p.tokens = (int64_t)a->batch * a->L;
  const int heads = a->q_heads + a->kv_heads;
  if (p.tokens == 0 || heads == 0) return VB_OK;
  VB_REQUIRE(a->positions && (!a->q_heads || (a->q && a->q_out)) &&
                 (!a->kv_heads || (a->k && a->k_out)),
             "vb_rotate_axes: null tensor");
  p.positions = a->positions;
  p.L = a->L; p.dim = a->dim; p.eps = a->eps;
  int64_t odd = 0;
  bool same = true;
  for (int i = 0; i < 2; ++i) {
    p.heads[i] = i ? a->kv_heads : a->q_heads;
    p.src[i] = i ? a->k : a->q;
    p.dst[i] = i ? a->k_out : a->q_out;
    p.norm[i] = p.heads[i] ? (i ? a->k_norm : a->q_norm) : nullptr;
    if (!p.heads[i]) continue;
    VB_REQUIRE((uintptr_t)p.src[i] % 2 == 0 && (uintptr_t)p.dst[i] % 2 == 0 &&
                   (uintptr_t)p.norm[i] % 2 == 0,
               "vb_rotate_axes: odd address");
    odd |= (int64_t)((uintptr_t)p.src[i] / 2) | (int64_t)((uintptr_t)p.dst[i] / 2) |
           (int64_t)((uintptr_t)p.norm[i] / 2);
    same = same && p.src[i] == p.dst[i] && !p.norm[i];
    for (int k = 0; k < 3; ++k) {
      p.s_in[i][k] = i ? a->k_strides[k] : a->q_strides[k];
      p.s_out[i][k] = i ? a->k_out_strides[k] : a->q_out_strides[k];
      odd |= p.s_in[i][k] | p.s_out[i][k];
      same = same && p.s_in[i][k] == p.s_out[i][k];
    }
  }
  p.keep = same;
  // Tokens of a CTA: up to 32, fewer while that leaves SMs without work.
  int per = RT_TABLE / p.half < RT_TOKENS ? RT_TABLE / p.half : RT_TOKENS;
  if (per > p.tokens / 592) per = (int)(p.tokens / 592);
  p.per = per > 1 ? per : 1;
  p.groups = (a->L + p.per - 1) / p.per;
  const int64_t ctas = (int64_t)p.groups * a->batch;
  VB_REQUIRE(ctas <= 0x7fffffffll, "vb_rotate_axes: too many tokens");
  const bool vec = odd % 8 == 0;
  cudaStream_t s = as_stream(stream);
  const int lpr = a->dim > 128 ? 16 : a->dim > 64 ? 8 : 4;
  if (lpr == 16) rt_launch<16>(p, (unsigned)ctas, vec, s);
  else if (lpr == 8) rt_launch<8>(p, (unsigned)ctas, vec, s);
  else rt_launch<4>(p, (unsigned)ctas, vec, s);
  return check_launch("rotate_kernel");
}
