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
constexpr int RT_TABLE = 1024;     // (token, pair) sines and cosines of a CTA
constexpr int RT_AHEAD = 4;        // rows that a thread has in flight

struct RotateParams {
  const uint16_t *src[2];          // q, k
  uint16_t *dst[2];
  const uint16_t *norm[2];
  int64_t s_in[2][3], s_out[2][3]; // element strides of batch, head, row
  const int32_t *positions;        // [axes][tokens]
  int64_t tokens;                  // batch * L
  int L, heads[2], dim, half, per; // per: tokens of a CTA
  float eps;
  bool keep;                       // dims from R on are in place already
  double turns[RT_PAIRS];          // frequency / 2 pi
  uint8_t axis[RT_PAIRS];
};

__device__ __forceinline__ void rt_load(float (&x)[8], const uint16_t *p, bool vec) {
  uint32_t w[4];
  if (vec) {
    const uint4 v = ldg_v4(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = p[2 * j] | ((uint32_t)p[2 * j + 1] << 16);
  }
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
// others 16 dims that only the norm changes. A CTA makes the sines of its tokens
// and then goes through their rows, all heads of a token one after another.
template <int LPR, bool NORM>
__global__ void __launch_bounds__(RT_THREADS) rotate_kernel(const __grid_constant__ RotateParams p,
                                                            bool vec) {
  __shared__ float2 s_cs[RT_TABLE];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, heads = p.heads[0] + p.heads[1];
  const int64_t t0 = (int64_t)blockIdx.x * p.per;
  const int n = (int)min((int64_t)p.per, p.tokens - t0);
  const int j = tid % LPR, turned = p.half >> 3;
  // dims of this lane: two runs of eight
  const int d0 = j < turned ? j * 8 : 2 * p.half + (j - turned) * 16;
  const int d1 = j < turned ? p.half + j * 8 : d0 + 8;
  const bool live = j * 16 < p.dim && !(p.keep && j >= turned);
  constexpr int STEP = RT_THREADS / LPR;
  const int rows = n * heads;
  bool ready = false;
  for (int r0 = tid / LPR; r0 - tid / LPR < rows; r0 += STEP * RT_AHEAD) {
    float a[RT_AHEAD][8], b[RT_AHEAD][8];
#pragma unroll
    for (int k = 0; k < RT_AHEAD; ++k) {
      const int r = r0 + k * STEP;
      if (r < rows && live) {
        const int t = r / heads, hh = r - t * heads, kind = hh >= p.heads[0];
        const int h = kind ? hh - p.heads[0] : hh;
        const int64_t at = t0 + t, bb = at / p.L, i = at - bb * p.L;
        const uint16_t *src = p.src[kind] + bb * p.s_in[kind][0] + h * p.s_in[kind][1] +
                              i * p.s_in[kind][2];
        rt_load(a[k], src + d0, vec);
        rt_load(b[k], src + d1, vec);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[k][e] = b[k][e] = 0.f;
      }
    }
    if (!ready) {  // while the first rows are on their way
      for (int x = tid; x < n * p.half; x += RT_THREADS) {
        const int t = x / p.half, i = x - t * p.half;
        const double turn = p.positions[p.axis[i] * p.tokens + t0 + t] * p.turns[i];
        float2 cs;
        sincospif(2.f * (float)(turn - rint(turn)), &cs.y, &cs.x);
        s_cs[x] = cs;
      }
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int k = 0; k < RT_AHEAD; ++k) {
      const int r = r0 + k * STEP;
      const int t = r / heads, hh = r - t * heads, kind = hh >= p.heads[0];
      if constexpr (NORM) {
        const uint16_t *w = p.norm[kind];
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(a[k][e], a[k][e], fmaf(b[k][e], b[k][e], ss));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && live) {
          const float inv = rsqrtf(ss / p.dim + p.eps);
          float wa[8], wb[8];
          rt_load(wa, w + d0, vec);
          rt_load(wb, w + d1, vec);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a[k][e] *= inv * wa[e];
            b[k][e] *= inv * wb[e];
          }
        }
      }
      if (r >= rows || !live) continue;
      if (j < turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 cs = s_cs[t * p.half + j * 8 + e];
          const float x = a[k][e], y = b[k][e];
          a[k][e] = fmaf(x, cs.x, -y * cs.y);
          b[k][e] = fmaf(y, cs.x, x * cs.y);
        }
      }
      const int h = kind ? hh - p.heads[0] : hh;
      const int64_t at = t0 + t, bb = at / p.L, i = at - bb * p.L;
      uint16_t *dst = p.dst[kind] + bb * p.s_out[kind][0] + h * p.s_out[kind][1] +
                      i * p.s_out[kind][2];
      rt_store(dst + d0, a[k], vec);
      rt_store(dst + d1, b[k], vec);
    }
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
                 a->q_heads <= 1 << 20 && a->kv_heads <= 1 << 20,
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
  // Tokens of a CTA: as many as give each thread a full turn of rows, fewer while that
  // leaves SMs without work.
  const int lpr = a->dim > 128 ? 16 : a->dim > 64 ? 8 : 4;
  int per = RT_THREADS / lpr * RT_AHEAD / heads;
  per = per < RT_TABLE / p.half ? per : RT_TABLE / p.half;
  if (per > p.tokens / 296) per = (int)(p.tokens / 296);
  p.per = per > 1 ? per : 1;
  const int64_t ctas = (p.tokens + p.per - 1) / p.per;
  VB_REQUIRE(ctas <= 0x7fffffffll, "vb_rotate_axes: too many tokens");
  const bool vec = odd % 8 == 0;
  cudaStream_t s = as_stream(stream);
  if (lpr == 16) rt_launch<16>(p, (unsigned)ctas, vec, s);
  else if (lpr == 8) rt_launch<8>(p, (unsigned)ctas, vec, s);
  else rt_launch<4>(p, (unsigned)ctas, vec, s);
  return check_launch("rotate_kernel");
}
