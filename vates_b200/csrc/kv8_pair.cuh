// Tensor-core products of a pair of CTAs (tcgen05 cta_group::2) over the paged
// 8-bit cache: operands, barriers and issue, shared by the kernels that use them.
#pragma once

#include "kv8_attn.cuh"
#include "tc100.cuh"

namespace vb {
namespace {

constexpr int KP_BLOCK = 16384;         // 128 rows x 64 f16, 128-byte swizzle
constexpr uint64_t KP_WAIT_NS = 2000000000ull;

// Byte offset of 16-byte chunk c of row r in a 128-row x 64-column block.
__device__ __forceinline__ uint32_t kp_sw(int r, int c) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}
__host__ __device__ constexpr uint32_t kp_idesc(int N, bool b_mn) {  // f16 x f16 -> f32, M = 256
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(256 >> 4) << 24);
}
// 16 codes of chunk ch -> two 16-byte chunks of f16 in row r of a tile (`block` bytes for
// each 64 columns); neighbouring blocks store them in opposite order so that the eight
// lanes of a store pass hit all banks.
__device__ __forceinline__ void kp_store_codes(const uint4 &x, uint8_t *tile, int block, int r,
                                               int ch) {
  const int e0 = (ch >> 2) & 1, c = 2 * (ch & 3);
  const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u,
                         x.w ^ 0x80808080u};
  uint4 o[2];
  o[0] = make_uint4(h2_codes(__byte_perm(w[0], 0x64646464u, 0x4140)),
                    h2_codes(__byte_perm(w[0], 0x64646464u, 0x4342)),
                    h2_codes(__byte_perm(w[1], 0x64646464u, 0x4140)),
                    h2_codes(__byte_perm(w[1], 0x64646464u, 0x4342)));
  o[1] = make_uint4(h2_codes(__byte_perm(w[2], 0x64646464u, 0x4140)),
                    h2_codes(__byte_perm(w[2], 0x64646464u, 0x4342)),
                    h2_codes(__byte_perm(w[3], 0x64646464u, 0x4140)),
                    h2_codes(__byte_perm(w[3], 0x64646464u, 0x4342)));
  uint8_t *base = tile + (ch >> 2) * block;
  *reinterpret_cast<uint4 *>(base + kp_sw(r, c + e0)) = e0 ? o[1] : o[0];
  *reinterpret_cast<uint4 *>(base + kp_sw(r, c + 1 - e0)) = e0 ? o[0] : o[1];
}
// The pair's products, issued by one thread of CTA 0: rows 0-127 of A and D are
// CTA 0's, 128-255 CTA 1's; each holds half of B's N. The whole warp comes here
// (its values are then uniform); `one` is true in the lane that issues.
__device__ __forceinline__ uint32_t kp_elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(r));
  return r;
}
__device__ __forceinline__ void kp_mma_ss(uint32_t one, uint32_t d_tmem, uint64_t adesc,
                                          uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
      : "memory");
}
// Arrive on this barrier of both CTAs once all products issued so far are done.
__device__ __forceinline__ void kp_commit(uint32_t one, uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster"
      ".b64 [%0], %1;\n}\n" ::"r"(tc::smem_u32(bar)),
      "h"((uint16_t)3), "r"(one)
      : "memory");
}
// Arrive on CTA 0's barrier, from either CTA. What the arrival stands for is
// ordered before it on its own SM: operands in shared memory by the proxy fence,
// P and O in TMEM by tcgen05.wait. A release of cluster scope in its place costs
// about 1,300 cycles an arrival.
__device__ __forceinline__ void kp_arrive_leader(uint64_t *bar) {
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n"
      " mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(tc::smem_u32(bar))
      : "memory");
}
// Relaxed: nothing of what a thread has written to global memory needs to be there
// for the other CTA, and waiting for it cost most of a microsecond.
__device__ __forceinline__ void kp_cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void kp_cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void kp_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void kp_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

}  // namespace
}  // namespace vb
