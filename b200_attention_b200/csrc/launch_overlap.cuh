// Launches whose start overlaps the end of the kernel before them in the stream (programmatic dependent launch): the
// grid may be brought up once every block of the previous kernel has called launch_dependents() or ended, and its
// threads stop in wait_for_previous() until that kernel has completed and its memory is visible. A kernel launched this
// way calls both, the latter before its first access to anything that an earlier kernel may read or write.
#pragma once

#include <utility>

#include <cuda_runtime.h>

namespace b200attn {

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

template <class... Params, class... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream,
                              Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace b200attn
