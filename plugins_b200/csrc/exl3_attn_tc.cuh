// exl3_attn_tc.cuh -- the tensor-core pieces the paged attention kernels share (sm_100a): packed f32 arithmetic, bounded
// mbarrier waits, TMA boxes of the cache's pages, operand descriptors, and MMAs issued by one elected lane.
#pragma once
#include <cuda.h>
#include <stdint.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_tc.cuh"

namespace exl3 {

// The layer's K or V, and the queries, as tensor maps (exl3_attn_tc.cu).
bool kv_tensor_map(CUtensorMap& map, void* base, const AttnParams& p, int dim, int tile_keys);
bool q_tensor_map(CUtensorMap& map, const AttnParams& p, int dim, int tokens);

namespace tc {

// Two f32 in one 64-bit register pair: one issue slot for both.
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// the largest of three (NaN is passed over: it shows in its own probability)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bounded wait (about two seconds) that also gives up when another role has.  The abort flag and the clock are read once
// in many polls: a read of the global timer between polls held each wait up, and every tile's chain has three of them
// (32 x 16-token trees 207 us with it, 192 without).
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* err) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) != 0u) continue;
    if (*abort_flag) return false;
    if ((i & 1023u) != 0u) continue;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    else if (now - t0 > 2000000000ull) {
      *abort_flag = 1u;
      atomicOr(err, kErrWaitTimeout);
      return false;
    }
  }
}

// A box of the cache: 64 columns from x, the rows from `tok` of one page and head.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int tok, int head, int page,
                                        uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(tok), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// Shared-memory descriptor of an operand whose rows are k (keys) and whose contiguous direction is M or N: 64-element
// blocks of 128-byte swizzled rows, `block_bytes` apart; 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t block_bytes) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((block_bytes >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// Instruction descriptor of kind::f16 with f32 accumulators; b_mn: B's contiguous direction is N.
template <bool BF16>
constexpr uint32_t attn_idesc(int m, int n, bool b_mn) {
  return umma_idesc(m, n) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// The MMA warp runs converged and one elected lane issues: its operands then stay in uniform registers.  (Issued inside
// a one-lane branch, each MMA took some 100 clocks to issue, against the 64 it runs for: 4.1k clocks per 256 x 128 tile.)
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}
// The same value, known to the compiler to be one for the whole warp.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }
// A descriptor `bytes` further on (its address field counts 16 bytes in the low word).
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t lo_add) {
  return (desc & 0xFFFFFFFF00000000ull) | (static_cast<uint32_t>(desc) + lo_add);
}
// D[tmem] (+)= A[smem] * B[smem]^T, where `on`
__device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], where `on`
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// Arrives on `bar` when every tcgen05 operation the elected lane issued before has completed.
__device__ __forceinline__ void commit(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}

// Orders uses of registers loaded by tmem_ld32 after an earlier wait (tmem_wait_ld of another load).
__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

}  // namespace tc
}  // namespace exl3
