// What kernels on pairs of SMs share (`cta_group::2`): PTX wrappers, arrivals and waits between the two CTAs of a cluster.
#pragma once
#include "gemm_common.cuh"

namespace ogb {

// ------------------------------------------------------------------------------- pair forms of the PTX wrappers
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// into this CTA's shared memory, counted on the barrier at the cluster address `bar`
__device__ __forceinline__ void pair_tma_load_2d(void* smem_dst, const CUtensorMap* m, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void pair_umma_f16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the barrier at this offset in both CTAs once every MMA issued so far is done
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(smem_u32(bar)), "h"(uint16_t(3)) : "memory");
}
// bar: cluster address.  The arrival names no scope, so what PTX promises is a release to the arriving CTA, while the waiter of the second CTA's arrivals is in
// the first one: the text of the memory model does not order them.  What this rests on: the data concerned are the arriving CTA's own shared memory, whose
// writers have each passed the proxy fence (which completes their stores) before their warp arrives, and its tensor memory, whose reads are complete after
// tcgen05.wait; no cache lies between them and the tensor core that the arrival releases.  Arrivals of the scope of the cluster, all of them or relayed by one
// warp of the second CTA, would be ordered by the text too and cost (us, none / all / relayed): the int4 product of 777 tokens at the head of gemm_pair.cu
// 77 / 115 / 107, MXFP4 6000 rows of 32 experts, 5760 x 2880 178 / 277 / 266.
__device__ __forceinline__ void cluster_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool cluster_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// mbar_wait_bounded for barriers on which the other CTA arrives
__device__ __forceinline__ bool cluster_wait_bounded(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns = 2000000000ull) {
  uint64_t t0 = 0;
  uint32_t spins = 0;
  while (!cluster_try_wait(bar, parity)) {
    if ((++spins & 0x3ff) == 0) {
      if (*abort_flag) return false;
      const uint64_t now = global_timer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > timeout_ns) return false;
    }
  }
  return true;
}

}  // namespace ogb
