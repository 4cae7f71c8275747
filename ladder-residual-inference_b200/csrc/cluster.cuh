// Thread-block clusters: addresses in another CTA's shared memory, the cluster barrier, and what kernels on pairs of SMs (cta_group::2) share.  Such a kernel is kept off by LRI_ONE_SM and
// by option gemm_pair = 0, and takes no sums of one or two K steps: gemm_pair.cu says why.
#pragma once

#include "tcgen05.cuh"

namespace lri {
namespace tc {

// an address of this CTA's shared memory in the CTA of this rank
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// The barrier of all threads of a cluster, in its two halves.  Its .aligned forms are a warp's, not a thread's: lanes that come one by one, out of a
// polling loop or from behind a branch that some took, have to meet first.  So both halves begin by that.
__device__ __forceinline__ void cluster_arrive_relaxed() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// publishes what was written before it
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- pairs of SMs -----------------------------------------------------------------------------------------------------------------
// `bar` may lie in either CTA of the pair
__device__ __forceinline__ void tma_load_pair(uint32_t smem_dst, const CUtensorMap* tmap, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_dst), "l"(tmap), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// arrives on the barrier at this offset in both CTAs
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
// publishes what was written before it
__device__ __forceinline__ void arrive_and_publish(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

}  // namespace tc
}  // namespace lri
