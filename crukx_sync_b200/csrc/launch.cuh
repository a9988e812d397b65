// Kernels that follow one another closely: the second is set up while the first still runs and waits
// for its memory at after_previous() (programmatic dependent launch).  Only for a kernel launched
// directly behind another one of the same call.
#pragma once

#include <cuda_runtime.h>

namespace crx {

// Everything the kernels before wrote is here from this point on.  (At once in a kernel that was
// launched the ordinary way.)
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The next kernel may be set up as soon as every CTA has come to this.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... Params, class... Args>
cudaError_t launch_behind(void (*kernel)(Params...), unsigned grid, unsigned block, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace crx
