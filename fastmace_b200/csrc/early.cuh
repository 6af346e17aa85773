// A launch behind another of this library's: its CTAs come to the SMs while the one before still runs, and wait there (kernels_before)
// for all that it has written. The launch's time, about 1.5 us, is hidden where the one before has said that it may be (let_next_come).
#pragma once

#include "fmb_common.cuh"

namespace fmb {

// Ahead of the first read or write of global memory. What is read of what the kernels before have written is read by way of pointers that have
// been named here: the compiler takes a load of what a kernel never writes (__ldg, const __restrict__) for one that may come at any time, and
// could move it before the wait, but not before its address is there.
template <typename... Pointers>
__device__ __forceinline__ void kernels_before(Pointers&... pointers) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    ((void)([&] { asm volatile("" : "+l"(pointers) : : "memory"); }()), ...);
}
// once every CTA of a launch has said so, the next one's may come
__device__ __forceinline__ void let_next_come() { asm volatile("griddepcontrol.launch_dependents;"); }

template <typename... Parameters, typename... Arguments>
cudaError_t launch_early(void (*kernel)(Parameters...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const Arguments&... arguments) {
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, Parameters(arguments)...);
}

}  // namespace fmb
