// Kernels that may start beside the one in front of them in their stream (programmatic dependent launch): launch,
// barrier set-up and first instructions fall under that one's end.  Such a kernel touches no memory before wait_previous(),
// which all of its threads call, so that what comes behind it comes behind both.  What it reads may be written while
// it lives already, so it reads by ordinary loads: a read-only one (__ldg) might find a line that was fetched before.
#pragma once
#include "common.cuh"

namespace ifv2 {

__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// beside: the kernel may start while the one in front of it still runs.
template <typename... Params, typename... Args>
cudaError_t launch_kernel(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, bool beside, const Args&... args) {
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}
template <typename... Params, typename... Args>
cudaError_t launch_beside(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  return launch_kernel(kernel, grid, threads, smem, stream, true, args...);
}

}  // namespace ifv2
