// pdl.cuh — programmatic stream serialisation shared by the small kernels: each waits for the
// previous kernel of its stream before it touches memory and lets the next one launch at once.
#pragma once
#include <cuda_runtime.h>

#include "sm100.cuh"

namespace fbfp {

__device__ __forceinline__ void pdl_prologue() {
  sm100::grid_dependency_wait();
  sm100::grid_launch_dependents();
}

// Launch with programmatic stream serialisation.
template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace fbfp
