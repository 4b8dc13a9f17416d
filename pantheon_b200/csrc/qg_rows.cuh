// qg_rows.cuh -- stores of accumulator rows.  An epilogue warp has a row per lane
// (TMEM's layout), so a lane's 16-byte stores meet 31 other rows in one
// instruction: 32 lines, a clock each.  Exchanged among four (eight) neighbouring
// lanes first, each instruction writes 64 (128) contiguous bytes of eight (four)
// rows instead.  And reads of other CTAs' partial rows over distributed shared memory.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace qg {

__device__ __forceinline__ uint4 shfl_xor_u4(uint4 v, int mask) {
    return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, mask), __shfl_xor_sync(0xffffffffu, v.y, mask),
                      __shfl_xor_sync(0xffffffffu, v.z, mask), __shfl_xor_sync(0xffffffffu, v.w, mask));
}

// N x N transpose of 16-byte pieces among groups of N neighbouring lanes: v[j] of
// lane q becomes what was v[q] of lane j.  The whole warp calls it.
template <int N>
__device__ __forceinline__ void transpose_lanes(uint4 (&v)[N]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 1; m < N; m *= 2) {
        const bool high = lane & m;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((i & m) == 0) {
                const uint4 got = shfl_xor_u4(high ? v[i] : v[i + m], m);
                if (high) v[i] = got;
                else v[i + m] = got;
            }
    }
}

// 16 x 16 transpose of words among 16 neighbouring lanes.  The whole warp calls it.
__device__ __forceinline__ void transpose_words(uint32_t (&w)[16]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 1; m < 16; m *= 2) {
        const bool high = lane & m;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((i & m) == 0) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? w[i] : w[i + m], m);
                if (high) w[i] = got;
                else w[i + m] = got;
            }
    }
}

// The warp's 32 rows x 16 N bytes (lane l: row l): rows row0 + l below `rows`, from
// element `n0` (of `elem` bytes) on of rows of `cols` elements.  `vec`: rows and
// n0 start on 16 bytes and cols is a multiple of 16 bytes.  Without it a row's 64
// bytes go as 16 words of neighbouring lanes (two-byte elements at an odd place one by
// one), two rows per instruction: the MXFP4 product 4096x5004x2048 in bf16 takes 25.7 us
// and 4096x5001x2048 32.1, against 102 with each lane storing its pieces' elements
// one by one and 22.4 for 5000 columns.  `out` is aligned to its elements.  The whole
// warp calls it.
template <typename E, int N>
__device__ __forceinline__ void store_rows(E* out, int row0, int rows, int n0, int cols, bool vec, uint4 (&v)[N]) {
    const int lane = threadIdx.x & 31;
    if (vec) {
        constexpr int PER = 16 / sizeof(E);
        transpose_lanes(v);
        const int n = n0 + (lane % N) * PER;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = row0 + (lane & ~(N - 1)) + j;
            if (r < rows && n < cols) *reinterpret_cast<uint4*>(out + (size_t)r * cols + n) = v[j];
        }
    } else {
        constexpr int PER = 4 / sizeof(E);
#pragma unroll
        for (int part = 0; part < N / 4; ++part) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 t = v[4 * part + i];
                w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
            }
            transpose_words(w);
            const int n = n0 + (16 * part + (lane & 15)) * PER;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = row0 + (lane & 16) + i;
                if (r >= rows || n >= cols) continue;
                E* dst = out + (size_t)r * cols + n;
                if constexpr (sizeof(E) == 4) {
                    *dst = w[i];
                } else if (n + 1 < cols && ((uintptr_t)dst & 3) == 0) {
                    *reinterpret_cast<uint32_t*>(dst) = w[i];
                } else {
                    dst[0] = (E)w[i];
                    if (n + 1 < cols) dst[1] = (E)(w[i] >> 16);
                }
            }
        }
    }
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

} // namespace qg
