// Thread-block clusters: addresses in another CTA's shared memory, and the cluster barrier.
#pragma once

#include "common.cuh"

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

}  // namespace tc
}  // namespace lri
