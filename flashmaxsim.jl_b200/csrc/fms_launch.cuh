// fms_launch.cuh -- launches that overlap the start of a kernel with the end of the one
// before it in the stream (programmatic dependent launch).  A kernel so launched calls
// dependency_wait() before it reads or writes global memory: it returns when everything
// the earlier kernel wrote is there.  Right after it the kernel lets the next one begin in
// the same way, which then takes the SMs as they fall free; about 2 us a launch.
//
// Such a kernel reads global memory by ordinary loads only: a load through the read-only
// path (__ldg, ld.global.nc) is for memory that nobody writes while the kernel runs, and
// this one runs already while the earlier one writes.
#pragma once
#include <cuda_runtime.h>

#include <utility>

namespace fms {

__device__ __forceinline__ void dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, std::forward<A>(args)...);
}

}  // namespace fms
