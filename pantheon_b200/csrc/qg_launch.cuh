// qg_launch.cuh -- launches that may begin under the tail of the kernel ahead
// on their stream (programmatic dependent launch), as clusters where asked.
#pragma once

#include "qg_common.cuh"

#include <utility>

namespace qg {

// A kernel launched by launch_overlapped calls this in every thread after its
// prologue and before its first access to global memory: it returns when all
// the kernels ahead are complete and their writes visible.  Then the next
// kernel may be launched.  That takes effect only once every CTA of this grid
// has asked for it, so all of them are resident and hold their tensor memory:
// CTAs of the next grid can delay none of them.
__device__ __forceinline__ void wait_previous_grid() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Loads of what the kernel ahead may have written, for after wait_previous_grid():
// spelled out, because the non-coherent path (`__ldg`, and what the compiler may make
// of a const pointer that nothing here writes through) is for memory that stays as it
// is while the kernel lives, and this kernel lives from under its predecessor's tail
// on.  `volatile` keeps them behind the wait; several in a row are still in flight at once.
__device__ __forceinline__ uint4 load_global(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_global(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_global(const uint16_t* p) {
    uint16_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_global(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

template <typename... KArgs, typename... Args>
inline cudaError_t launch_overlapped(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                     unsigned cluster, Args&&... args) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = block;
    lc.dynamicSmemBytes = smem;
    lc.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {cluster, 1, 1};
    lc.attrs = at;
    lc.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, kernel, std::forward<Args>(args)...);
}

} // namespace qg
