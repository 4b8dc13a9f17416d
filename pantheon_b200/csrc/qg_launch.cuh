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
