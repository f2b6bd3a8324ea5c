// Programmatic dependent launch for the kernels of a decoding step: each lets
// the next kernel on the stream start its prologue (barriers, TMEM, tensor
// maps) while it runs, and waits for the kernels before it, all their writes
// visible, before it touches global memory.  Every thread of every CTA waits,
// so a kernel's end implies the end of all kernels before it.
#pragma once

#include <cuda_runtime.h>

namespace vq {
namespace pdl {

__device__ __forceinline__ void trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Kernel F in clusters of `cluster` CTAs.  Dependent (over the kernels before
// it): for short kernels, where it saves about 0.8 us a call in a row of them;
// long ones gain nothing, and prompts' appends lost 5 %.
template <auto F, bool DEPENDENT = true, typename... A>
static inline bool launch(unsigned grid, unsigned threads, size_t smem, cudaStream_t st, int cluster,
                          const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (DEPENDENT) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster, at[n].val.clusterDim.y = 1, at[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, F, args...) == cudaSuccess;
}

}  // namespace pdl
}  // namespace vq
