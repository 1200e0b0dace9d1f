// Launches of one call that follow one another: the next one's CTAs may take their places on the SMs while the last is still running,
// and wait there for its end, which hides most of what lies between two launches (about 2 us).
#pragma once

#include <cuda_runtime.h>

namespace m2d {

// In the kernel that is followed, at its start: no CTA of the next is placed before all of this one's have started.
__device__ __forceinline__ void let_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// In the kernel that follows, before it reads what the last has written or writes what that reads; every thread calls it, so that
// whatever comes after this kernel comes after the last one too.  (In any other launch it does nothing.)  What the last kernel has written
// is read by plain loads: those of data declared read-only may be moved to before the wait.
__device__ __forceinline__ void follow_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
inline bool launch_following(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kern, args...) == cudaSuccess || (cudaGetLastError(), false);
}

}  // namespace m2d
