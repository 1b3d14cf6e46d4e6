// Sums over a CTA and the start of a cluster, for the losses' kernels (logits.cu, preference.cu).
#pragma once

#include <cuda_runtime.h>

namespace tiso {

// The sum of v over the CTA in a fixed order (thread 0 has it). shared: 32 numbers.
__device__ __forceinline__ double block_sum(double v, double* shared) {
  for (int d = 16; d; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < blockDim.x / 32 ? shared[threadIdx.x] : 0.0;
  if (threadIdx.x < 32)
    for (int d = 16; d; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
  __syncthreads();
  return v;
}

// The CTAs of a cluster write to one another's shared memory once, at their joins. Before that each
// has to have started: every thread says that its CTA has (and nothing about memory: relaxed), and
// waits for the others' ahead of the write.
__device__ __forceinline__ void cluster_started(int ctas) {
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void wait_for_start() {
  asm volatile("barrier.cluster.wait;" ::: "memory");
}

}  // namespace tiso
