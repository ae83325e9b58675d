// A launch that begins while the one before it in the stream is still at work: what a kernel sets up for itself, and the way to its first
// instruction, are then not on the way of the data.  let_next(): the next kernel's blocks may come as there is room; wait_before(): what the
// kernel before wrote is there.  Both do nothing in a kernel that was launched, or is followed, the ordinary way.  Every kernel that is
// launched so waits before it ends, so that the end of one is the end of all before it.
#pragma once

#include <cuda_runtime.h>

namespace nb200 {
namespace {

__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kern)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = a;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kern, args...);
}

}  // namespace
}  // namespace nb200
