// qg_mxfp4_mma.cuh -- the block-scaled e2m1 tensor-core product of the MXFP4 kernels.
#pragma once

#include "qg_ptx.cuh"

namespace qg {
namespace mx {

// tcgen05.mma kind::mxf4 (e2m1 x e2m1, ue8m0 per 32 along K) -> fp32.
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
        : "memory");
}

// Instruction descriptor with the scale ids (byte pair 0-1 or 2-3 of a scale word).
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t M, uint32_t N, uint32_t sf_id) {
    return make_idesc_bs(/*e2m1*/ 1, /*e2m1*/ 1, /*ue8m0*/ 1, M, N) | (sf_id << 4) | (sf_id << 29);
}

// Arrive on an mbarrier of the cluster without release: for handing over TMEM
// contents, complete after tcgen05.wait and ordered by the tcgen05 fences on
// both sides.  Not for shared or global memory.
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// One commit that arrives on the same barrier of both CTAs of a pair (the commit of
// this thread's products; pair `pair` of the cluster).
__device__ __forceinline__ void umma_commit_both(uint64_t* bar, uint32_t pair = 0) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)(3u << (2 * pair))) : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// mbar_wait of a whole warp: true in every lane, or false in every lane.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, DeviceStatus* status,
                                          uint32_t site) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, site));
}

} // namespace mx
} // namespace qg
