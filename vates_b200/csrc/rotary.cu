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
//
// What bounds it: HBM, in and out once. 65,536 tokens of 16/2 heads of 256 (1.21 GB) take
// 244 us, 4.95 TB/s or 0.76 of a copy, 2 x 8,191 of 32/8 heads of 128 62 us for 336 MB
// (5.4 TB/s); issue slots are half used, and rows are read 512 bytes at a time. The rows
// of one decode step cost the launch, 4 us.
#include "common.cuh"

namespace vb {
namespace {

constexpr int RT_THREADS = 256;
constexpr int RT_PAIRS = 128;      // most rotated pairs of a row

struct RotateParams {
  const uint16_t *src[2];          // q, k
  uint16_t *dst[2];
  const uint16_t *norm[2];
  int64_t s_in[2][3], s_out[2][3]; // element strides of batch, head, row
  const int32_t *positions;        // [axes][tokens]
  int64_t tokens;                  // batch * L
  int L, heads[2], dim, half, per, groups;  // log2 of a CTA's tokens, CTAs of a sequence
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
__device__ __forceinline__ f2 rt_pair(uint32_t w) {
  return f2_make(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ void rt_pairs(f2 (&x)[4], const uint4 &v) {
  x[0] = rt_pair(v.x); x[1] = rt_pair(v.y); x[2] = rt_pair(v.z); x[3] = rt_pair(v.w);
}
__device__ __forceinline__ void rt_store(uint16_t *p, const f2 (&x)[4], bool vec) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    f2_split(x[j], a, b);
    w[j] = pack_bf2(a, b);
  }
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
// others 16 dims that only the norm changes. A CTA takes up to STEP = 256 / LPR
// tokens of one sequence, a power of two of them; its STEP rows at a time are those
// tokens of one head, or of several heads where it has fewer tokens. So a thread
// stays with one token: its sines are made once, and from head to head only a
// pointer moves.
// Rows of a thread in flight, and CTAs per SM: 2 and 4, with a norm, whose registers
// leave room for 3 CTAs, 3 and 3 (65,536 tokens of 16/2 heads of 256 with it 248 to 258 us
// a call, 306 the other way). Without it 2 x 8,191 of 32/8 heads of 128 take 64.5, and 59 to
// 61 with 3 and 3: the choice was made when a CTA took more tokens (79 and 83).
template <int LPR, bool NORM>
__global__ void __launch_bounds__(RT_THREADS, NORM ? 3 : 4) rotate_kernel(const __grid_constant__ RotateParams p,
                                                               bool vec) {
  constexpr int STEP = RT_THREADS / LPR, RT_AHEAD = NORM ? 3 : 2;
  __shared__ float2 s_cs[STEP * LPR * 8];  // [token][pair % 8][pair / 8]
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, j = tid % LPR, turned = p.half >> 3;
  const int b = blockIdx.x / p.groups, i0 = (blockIdx.x - b * p.groups) << p.per;
  const int n = min(1 << p.per, p.L - i0);
  const int t = (tid / LPR) & ((1 << p.per) - 1), h0 = (tid / LPR) >> p.per, h_step = STEP >> p.per;
  const int heads = p.heads[0] + p.heads[1];
  // dims of this lane: two runs of eight
  const int d0 = j < turned ? j * 8 : 2 * p.half + (j - turned) * 16;
  const int d1 = j < turned ? p.half + j * 8 : d0 + 8;
  const bool live = t < n && j * 16 < p.dim && !(p.keep && j >= turned);
  const int64_t in0 = b * p.s_in[0][0] + (i0 + t) * p.s_in[0][2];
  const int64_t in1 = b * p.s_in[1][0] + (i0 + t) * p.s_in[1][2] - p.heads[0] * p.s_in[1][1];
  uint4 x[RT_AHEAD], y[RT_AHEAD];
  auto fetch = [&](int h) {
#pragma unroll
    for (int k = 0; k < RT_AHEAD; ++k, h += h_step) {
      x[k] = y[k] = make_uint4(0, 0, 0, 0);
      if (h < heads && live) {
        const uint16_t *src = h < p.heads[0] ? p.src[0] + in0 + h * p.s_in[0][1]
                                             : p.src[1] + in1 + h * p.s_in[1][1];
        x[k] = rt_load(src + d0, vec);
        y[k] = rt_load(src + d1, vec);
      }
    }
  };
  fetch(h0);
  // sines while the first rows are on their way
  for (int z = tid; z < n * p.half; z += RT_THREADS) {
    const int u = z / p.half, i = z - u * p.half;
    const double turn = p.positions[p.axis[i] * p.tokens + (int64_t)b * p.L + i0 + u] * p.turns[i];
    float2 cs;
    sincospif(2.f * (float)(turn - rint(turn)), &cs.y, &cs.x);
    s_cs[u * p.half + (i & 7) * turned + (i >> 3)] = cs;
  }
  __syncthreads();
  f2 cs[4], sn[4];
  if (j < turned && t < n) {
    const float2 *e = s_cs + t * p.half + j;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = e[2 * k * turned], c = e[(2 * k + 1) * turned];
      cs[k] = f2_make(a.x, c.x);
      sn[k] = f2_make(a.y, c.y);
    }
  }
  const f2 minus = f2_make(-1.f, -1.f);
  const int64_t out0 = b * p.s_out[0][0] + (i0 + t) * p.s_out[0][2];
  const int64_t out1 = b * p.s_out[1][0] + (i0 + t) * p.s_out[1][2] - p.heads[0] * p.s_out[1][1];
  // (all lanes of a row, and of its warp, go through the same heads or one more)
  for (int h = h0; h - h0 < heads; h += h_step * RT_AHEAD) {
#pragma unroll
    for (int k = 0; k < RT_AHEAD; ++k) {
      const int hk = h + k * h_step;
      const bool q = hk < p.heads[0];
      f2 u[4], v[4];
      rt_pairs(u, x[k]);
      rt_pairs(v, y[k]);
      if constexpr (NORM) {
        const uint16_t *w = q ? p.norm[0] : p.norm[1];
        f2 s2 = f2_mul(u[0], u[0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e > 0) s2 = f2_fma(u[e], u[e], s2);
          s2 = f2_fma(v[e], v[e], s2);
        }
        float ss, s1;
        f2_split(s2, ss, s1);
        ss += s1;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && live) {
          const float inv = rsqrtf(ss / p.dim + p.eps);
          const f2 inv2 = f2_make(inv, inv);
          f2 wu[4], wv[4];
          rt_pairs(wu, rt_load(w + d0, vec));
          rt_pairs(wv, rt_load(w + d1, vec));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            u[e] = f2_mul(u[e], f2_mul(wu[e], inv2));
            v[e] = f2_mul(v[e], f2_mul(wv[e], inv2));
          }
        }
      }
      if (hk >= heads || !live) continue;
      if (j < turned) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f2 c = u[e], s = v[e];
          u[e] = f2_fma(c, cs[e], f2_mul(f2_mul(s, sn[e]), minus));
          v[e] = f2_fma(s, cs[e], f2_mul(c, sn[e]));
        }
      }
      uint16_t *dst = q ? p.dst[0] + out0 + hk * p.s_out[0][1] : p.dst[1] + out1 + hk * p.s_out[1][1];
      rt_store(dst + d0, u, vec);
      rt_store(dst + d1, v, vec);
    }
    fetch(h + h_step * RT_AHEAD);
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
    const int extent[3] = {a->batch, p.heads[i], a->L};
    for (int k = 0; k < 3; ++k) {
      VB_REQUIRE(extent[k] == 1 || (i ? a->k_out_strides[k] : a->q_out_strides[k]) != 0,
                 "vb_rotate_axes: rows of an output in one place (a stride of 0)");
      p.s_in[i][k] = i ? a->k_strides[k] : a->q_strides[k];
      p.s_out[i][k] = i ? a->k_out_strides[k] : a->q_out_strides[k];
      odd |= p.s_in[i][k] | p.s_out[i][k];
      same = same && p.s_in[i][k] == p.s_out[i][k];
    }
  }
  p.keep = same;
  // Tokens of a CTA (a power of two): as many as it has rows at a time, fewer as long as
  // there are fewer than 16 CTAs an SM, the last of which would keep few SMs busy (2 x 8,191
  // tokens of 32/8 heads of 128: 32, 16, 8, 4 and 2 tokens 80, 72, 66, 63 and 69 us), and
  // every thread still has all its rows in flight (4,096 tokens of 16/2 heads of 256: 8 tokens
  // 23 us, one 42); fewer than that where SMs would have none.
  const int lpr = a->dim > 128 ? 16 : a->dim > 64 ? 8 : 4;
  const int turn = RT_THREADS / lpr * (p.norm[0] || p.norm[1] ? 3 : 2);
  p.per = lpr == 16 ? 4 : lpr == 8 ? 5 : 6;
  while (p.per > 0 && (p.tokens >> p.per) < 148 * 16 && (int64_t)heads << p.per >= 2 * turn) --p.per;
  while (p.per > 0 && (p.tokens >> p.per) < 148 * 2) --p.per;
  p.groups = (a->L + (1 << p.per) - 1) >> p.per;
  const int64_t ctas = (int64_t)p.groups * a->batch;
  VB_REQUIRE(ctas <= 0x7fffffffll, "vb_rotate_axes: too many tokens");
  const bool vec = odd % 8 == 0;
  cudaStream_t s = as_stream(stream);
  if (lpr == 16) rt_launch<16>(p, (unsigned)ctas, vec, s);
  else if (lpr == 8) rt_launch<8>(p, (unsigned)ctas, vec, s);
  else rt_launch<4>(p, (unsigned)ctas, vec, s);
  return check_launch("rotate_kernel");
}
