// tcgen05 / TMEM / TMA building blocks shared by the tensor-core kernels (pointwise.cu, affine_bwd.cu):
// thin wrappers over the PTX, bounded waits, and the shared-memory matrix descriptor.
#pragma once

#include "dwbnq_fused.cuh"

namespace dwbnq {

constexpr unsigned long long kPwWaitNs = 2000000000ull;

// ---- sm_100a PTX wrappers ------------------------------------------------------------------

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *tm, int x, int y, unsigned long long *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(tm), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
// Bounded waits. Most of the twenty-odd warps of a CTA wait most of the time;
// the poll carries a suspend-time hint so that a waiting warp is parked by the hardware and
// leaves the issue slots to the warps that compute (a bare spin took about a third of them).
__device__ __forceinline__ bool pw_try_wait(unsigned long long *bar, unsigned int parity) {
  unsigned int ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool pw_wait_lane(unsigned long long *bar, unsigned int parity) {
  if (pw_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
#pragma unroll 1
  for (unsigned int i = 0; i < (1u << 28); ++i) {
    if (pw_try_wait(bar, parity)) return true;
    if (global_timer_ns() - t0 > kPwWaitNs) break;
  }
  return false;
}
// Warp-uniform form: every lane has seen the phase, or every lane gives up.
__device__ __forceinline__ bool pw_wait(unsigned long long *bar, unsigned int parity) {
  bool ok = pw_wait_lane(bar, parity);
  if (!__all_sync(0xffffffffu, ok)) {
    if (__any_sync(0xffffffffu, ok) && !ok) ok = pw_try_wait(bar, parity);
    ok = __all_sync(0xffffffffu, ok);
  }
  return ok;
}
// Whether a warp of the CTA is giving up (*abort_v): one answer for the whole warp, whose lanes may read the word at different times.
__device__ __forceinline__ bool pw_giving_up(volatile int *abort_v) { return __any_sync(0xffffffffu, *abort_v != 0); }
// (a & mask) | set as one instruction. A logic instruction takes one immediate: with both constants known the compiler needs two,
// so `set` has to come from a value it cannot see through (opaque_constant).
__device__ __forceinline__ unsigned int and_or(unsigned int a, unsigned int mask, unsigned int set) {
  unsigned int r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(set));
  return r;
}
__device__ __forceinline__ unsigned int opaque_constant(unsigned int v) {
  unsigned int r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// True in one lane of a converged warp. TMA and tcgen05 instructions take their operands from uniform registers: issued under this
// predicate from code the whole warp walks through, addresses and descriptors stay there; issued under `lane == 0` every
// operand is moved over one instruction at a time (the MMA thread of the weight gradient: 1400 cycles per four MMAs against 600).
__device__ __forceinline__ bool elect_one() {
  unsigned int ok;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void mbar_arrive(unsigned long long *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The barrier receives one arrival once every MMA this thread has issued so far is complete.
__device__ __forceinline__ void tc_commit(unsigned long long *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[128 x N] (+)= A[128 x 8] * B[N x 8]^T, TF32 operands from shared memory, fp32 accumulator in TMEM.
__device__ __forceinline__ void tc_mma_tf32(unsigned int tmem_d, unsigned long long da, unsigned long long db,
                                            unsigned int idesc, unsigned int accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Four consecutive elements as floats (16-byte load of fp32, 8-byte load of fp16).
__device__ __forceinline__ float4 pw_load4(const float *p) { return __ldg(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ float4 pw_load4(const __half *p) {
  const uint2 r = __ldg(reinterpret_cast<const uint2 *>(p));
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&r.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&r.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
// D[128 x N] (+)= A[128 x 16] * B[N x 16]^T, binary16 operands, fp32 accumulator.
__device__ __forceinline__ void tc_mma_f16(unsigned int tmem_d, unsigned long long da, unsigned long long db,
                                           unsigned int idesc, unsigned int accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 8 consecutive accumulator columns of this thread's lane (issue only; tc_ld_wait8 completes it).
__device__ __forceinline__ void tc_ld8(unsigned int taddr, unsigned int *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// Waits for this thread's outstanding TMEM loads. The loaded registers are operands, so the
// compiler cannot move a use of them above the wait.
__device__ __forceinline__ void tc_ld_wait8(unsigned int *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

// Shared-memory matrix descriptor of tcgen05.mma (addresses and offsets in bytes; the fields
// hold them divided by 16). layout 2 = 128-byte swizzle, 1 = 128-byte swizzle of 32-byte
// units, the only form the hardware takes for an MN-major operand of 32-bit elements.
__device__ __forceinline__ unsigned long long pw_smem_desc(unsigned int addr, unsigned int lbo, unsigned int sbo,
                                                          unsigned int layout) {
  return (unsigned long long)((addr >> 4) & 0x3fffu) | ((unsigned long long)((lbo >> 4) & 0x3fffu) << 16) |
         ((unsigned long long)((sbo >> 4) & 0x3fffu) << 32) | (1ull << 46) | ((unsigned long long)layout << 61);
}

}  // namespace dwbnq
