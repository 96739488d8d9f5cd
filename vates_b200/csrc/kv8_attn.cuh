// What the attention kernels over the paged 8-bit cache share.
#pragma once

#include "kv8.cuh"

namespace vb {

struct Kv8AttnParams {
  VbKv8Cache c;
  const uint16_t *q;
  int64_t qb, qh, ql;  // element strides of batch, head, row
  const int32_t *lens, *q_lens;
  uint16_t *out;
  float *lse;
  int32_t *status;
  // partial results of a key range: rows of float32 O, then (m, l) per row:
  // the range's weights are 2^(z - m), their sum l
  float *o_part;
  float2 *ml_part;
  // kv8_attn_kernel: a unit's first CTA and number of CTAs for the wide combine
  // kernel (`wide`), else a ticket word per unit, zero between calls
  int2 *units;
  uint32_t *tickets;
  bool wide;
  float scale_log2;  // scale * log2(e)
  int Hq, L, rep, len_add, causal, shift, vec;
  int row_tiles, splits;
  uint32_t rep_inv;  // floor(2^32 / rep) + 1
  // Segments in the place of sequences: (first sequence, sequences, first key, end):
  // all query rows of those sequences over the keys [first, end) that they have in
  // common, at most as far as each row sees. Another kernel joins their results, rows of
  // unnormalised O and (m, l): partial results as above, and for a unit that one CTA of
  // kv8_attn_kernel has whole, in o_res and ml_res.
  // The prefill kernel packs the rows that are there of a segment's sequences and leaves,
  // for the kernel that joins, its key ranges per row tile and the first row of every
  // sequence in places[0] and places[1 + sequence].
  const int4 *segs;
  int n_segs;
  int32_t *places;
  int pairs, longest;  // pairs of CTAs, key tiles of the longest segment
  int seg_lanes;       // lanes that count the rows of a segment: a power of two
  bool deal;           // segments of several row tiles: dealt by the rows that there are
  bool beside;       // runs beside the kernel ahead of it, of which it needs nothing
  float *o_res;
  float2 *ml_res;
  // Query row R (< 2^24) of the flattened (row, head of the group) order is
  // query R / rep: exact by one product while R * rep < 2^32.
  __device__ __forceinline__ int row_of(int R) const {
    return rep == 1 ? R : (int)__umulhi((uint32_t)R, rep_inv);
  }
};

// A row tile's share of the sequence: query row R of the flattened (row, head
// of the group) order is query R / rep, head R % rep, and sees the first
// visible(R / rep) keys.
struct Kv8Span {
  int keys, q_len, off, causal;
  __device__ int visible(int i) const {
    return i >= q_len ? 0 : causal ? max(0, off + i + 1) : keys;
  }
};

__device__ __forceinline__ Kv8Span kv8_span(const Kv8AttnParams &p, int b, bool flag) {
  Kv8Span s;
  int32_t *status = flag ? p.status : nullptr;
  const long long cap = (long long)p.c.max_pages * p.c.page;
  const long long keys = (long long)p.lens[b] + p.len_add;
  if (keys < 0 || keys > cap) flag_status(status, VB_STATUS_BOUNDS);
  s.keys = (int)min(max(keys, 0ll), cap);
  s.q_len = kv8_rows(p.q_lens, b, p.L, status);
  s.off = s.keys - s.q_len;
  s.causal = p.causal;
  return s;
}

// Keys of segment s that the rows of sequence b of it see, from its first key on.
__device__ __forceinline__ int kv8_reach(const int4 &s, int visible) {
  return max(0, min(visible, s.w) - s.z);
}
struct Kv8SegRow {
  int b, i, hr, vis;  // sequence, query, head of the group; keys seen (0: no such row)
};
// Query row R of a segment's flattened (sequence, row, head of the group) order.
__device__ __forceinline__ Kv8SegRow kv8_seg_row(const Kv8AttnParams &p, const int4 &s, int R) {
  const int per = p.L * p.rep, m = s.y == 1 ? R >= per : R / per, r = R - m * per;
  Kv8SegRow x;
  x.b = s.x + min(m, s.y - 1);
  x.i = p.row_of(r);
  x.hr = r - x.i * p.rep;
  x.vis = m < s.y ? kv8_reach(s, kv8_span(p, x.b, false).visible(x.i)) : 0;
  return x;
}

__device__ __forceinline__ float kv8_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Query values enter the products as f16 after a power of two that puts the
// row's largest one in [2^8, 2^9): exact for every bf16 down to 2^-23 of it.
// Returns the power (1 for a row with an infinity: that row is NaN anyway).
__device__ __forceinline__ float kv8_q_power(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) & 255;
  return __uint_as_float((uint32_t)(e == 255 ? 127 : min(254, 262 - e)) << 23);
}

// (The exponentials are shifted up before they are rounded to f16, whose
// largest value is 65504, so that a long tail of small weights is not flushed:
// the kernels' *_SHIFT. It cancels in O / l.)
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two codes + 128 in the low bytes of 0x64xx halves (1024 + 128 + code) minus
// 1152: exact f16 codes.
__device__ __forceinline__ uint32_t h2_codes(uint32_t magic) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(magic), "r"(0x64806480u));
  return r;
}

// 8 bf16 of a query row.
__device__ __forceinline__ uint4 kv8_load8(const uint16_t *q, bool vec) {
  if (vec) return ldg_v4(q);
  return make_uint4(q[0] | ((uint32_t)q[1] << 16), q[2] | ((uint32_t)q[3] << 16),
                    q[4] | ((uint32_t)q[5] << 16), q[6] | ((uint32_t)q[7] << 16));
}
// Two bf16 times the row's power of two, as f16.
__device__ __forceinline__ uint32_t kv8_q_h2(uint32_t w, float pw) {
  float lo, hi;
  f2_split(f2_mul(f2_make(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)),
                  f2_make(pw, pw)),
           lo, hi);
  return pack_h2(lo, hi);
}
// The lane's 8 bf16 of a row that LPR lanes hold together become f16 times the
// row's power of two, which is returned. Magnitudes of bf16 compare as integers.
template <int LPR>
__device__ __forceinline__ float kv8_q_scale(uint4 &v) {
  uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                        __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float pw = kv8_q_power(__uint_as_float(max(m << 16, m & 0xFFFF0000u)));
  v = make_uint4(kv8_q_h2(v.x, pw), kv8_q_h2(v.y, pw), kv8_q_h2(v.z, pw), kv8_q_h2(v.w, pw));
  return pw;
}

// Rows per row tile of the prefill kernel, and its launch (kv8_prefill.cu).
int kv8_prefill_rows();
int kv8_prefill_launch(const Kv8AttnParams &p, cudaStream_t s);
int kv8_prefill_launch_segments(const Kv8AttnParams &p, cudaStream_t s);

}  // namespace vb
