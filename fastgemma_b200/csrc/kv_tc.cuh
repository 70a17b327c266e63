// What the tcgen05 kernels over the KV cache share (kvtile.cu, kvaccum.cu):
// tiles of 128 query rows or slots, TMEM transfers, packed f32, masks as words.
#pragma once

#include <cuda_fp16.h>

#include "kv_attn.cuh"
#include "stream_ptx.cuh"
#include "tc_ptx.cuh"

namespace fgm {
namespace kv {

constexpr int kTM = 128;          // query rows per tile
constexpr int kTN = 128;          // slots per tile
constexpr int kChunk = 128 * 128; // bytes of one 128-byte column of Q or of a K tile

// Whether this is the warp's elected lane.  The warp that issues the MMAs runs
// as a whole, so that descriptors and counters stay in uniform registers, and
// elects a lane for the instructions of one thread.
__device__ __forceinline__ bool elected() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

__device__ __forceinline__ uint64_t desc128(uint32_t a) { return tc::sdesc_sw128(a); }

// D[tmem] (+)= A[tmem, f16] * B[smem desc, f16], f32 accumulate.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D f32, A and B f16, both K-major.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_st_x16(uint32_t a, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st_x8(uint32_t a, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

__device__ __forceinline__ void tmem_ld_x8(uint32_t a, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "r"(a));
}

__device__ __forceinline__ void tmem_ld_x2(uint32_t a, uint32_t (&r)[2]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(a));
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t (&r)[N]) {
  static_assert(N == 2 || N == 8, "widths in use");
  if constexpr (N == 8) tmem_ld_x8(a, r);
  else tmem_ld_x2(a, r);
}

// One row of results to global memory (bulk group of the thread).
__device__ __forceinline__ void bulk_s2g(void *dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(tc::smem_u32(src)), "r"(bytes)
               : "memory");
}

// Adds four f32 to memory, each rounded to nearest, without waiting.
__device__ __forceinline__ void red_add4(float4 *to, float4 v) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(v.x),
               "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// Orders plain accesses to global memory before later bulk copies.
__device__ __forceinline__ void fence_proxy_async_global() {
  asm volatile("fence.proxy.async.global;" ::: "memory");
}

__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Bits [a, b) of a 64-bit word, whatever a and b.
__device__ __forceinline__ uint64_t bit_range(int a, int b) {
  a = max(a, 0);
  b = min(b, 64);
  return a >= b ? 0 : (~0ull >> (64 - (b - a))) << a;
}

// Which of the positions t .. t + 31 a row sees: committed ones from `low` on,
// nodes by its words.
__device__ __forceinline__ uint32_t seen_from(int t, int len, int low, const uint64_t (&nodes)[4]) {
  uint32_t v = (uint32_t)bit_range(max(low, 0) - t, len - t);
  const int n = t - len;  // node of bit 0
  if (n > -32 && n < FGM_CUDA_TREE_MAX) {
    if (n < 0) {
      v |= (uint32_t)(nodes[0] << -n);
    } else {
      const int w = n >> 6, s = n & 63;
      v |= (uint32_t)(nodes[w] >> s);
      if (w < 3 && s > 32) v |= (uint32_t)(nodes[w + 1] << (64 - s));
    }
  }
  return v;
}

// Two f32 in one register pair: the packed forms of the FP32 pipe.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void split2(uint64_t d, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Waits until the phase with `parity` is over.  The tests put the warp to sleep
// for up to 10 us each: spinning, or reading a clock or the abort word between
// the tests, takes issue slots from the warps that work (256 nodes over 16K
// slots 65.7 us like this, 68.9 when the MMA warp alone spins, 71 when all do).
// After kWaitTests tests, two seconds asleep, the wait gives up and raises the
// abort word, on which later waits do not sleep any more: the loops run out,
// the CTA reports and leaves.
constexpr int kWaitTests = 200000;
__device__ __forceinline__ void wait_phase(uint64_t *bar, uint32_t parity, int *abort) {
  if (tc::mbar_try_wait(bar, parity)) return;
  uint32_t ok;
  for (int left = *(volatile int *)abort ? 1 : kWaitTests; left > 0; left--) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(tc::smem_u32(bar)), "r"(parity), "r"(10000u)
        : "memory");
    if (ok) return;
  }
  *(volatile int *)abort = 1;
}

}  // namespace kv
}  // namespace fgm
