// Programmatic dependent launch: a kernel's CTAs may start while the kernel before it on the stream still runs, and wait for its
// results where they need them.
#pragma once

#include "common.cuh"

namespace fp8gmm {

// Lets the next kernel of the stream start its CTAs as soon as all CTAs of this one have come here.
__device__ __forceinline__ void let_dependents_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Returns once the kernels before this one are complete and their writes visible; at once if it was launched the ordinary way.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches `kernel`; with `early` it may start before the kernel in front of it on the stream has ended.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), int grid, int threads, int smem, cudaStream_t s, bool early, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace fp8gmm
