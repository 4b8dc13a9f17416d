// qg_gated.cuh -- the activations of the gated products, and their slopes.
//
//   silu(g)      = g / (1 + exp(-g))
//   gelu_tanh(g) = 0.5 g (1 + tanh(z)) = g / (1 + exp(-2 z)),  z = sqrt(2/pi) (g + 0.044715 g^3)
// (0.5 (1 + tanh z) is the logistic function of 2 z), so both are g p with
// p = 1 / (1 + exp(-y)), and their slopes are p + g p (1 - p) dy/dg.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/pantheon_qgemm.h"

namespace qg {

// The logistic's argument of activation ACT: g, or 2 sqrt(2/pi) (1 + 0.044715 g^2) g.
template <int ACT>
__device__ __forceinline__ float gate_arg(float g) {
    if constexpr (ACT == QG_ACT_SILU) return g;
    else return g * fmaf(0.0713548162726f, g * g, 1.59576912161f);
}

// FAST: the hardware's 2^x and reciprocal, a few units in the last place of
// fp32, for results that are rounded to 16 bits or fewer.  exp(-y) reaches
// infinity at y = -88.7 and the quotient then is 0 (from 2^126 on with FAST,
// y = -87.3, where it is below 1.2e-38).
template <bool FAST>
__device__ __forceinline__ float logistic(float y) {
    if constexpr (FAST) return __fdividef(1.0f, 1.0f + __expf(-y));
    else return 1.0f / (1.0f + expf(-y));
}

template <int ACT, bool FAST>
__device__ __forceinline__ float gated(float g, float u) {
    return g * logistic<FAST>(gate_arg<ACT>(g)) * u;
}

// act(g) and its slope.  An infinite or huge g must not meet 1 - p = 0 (or p = 0) in
// a product, so the bend's argument is cut off where its factor p (1 - p) is exactly
// 0 in fp32 on either side: for silu beyond |g| = 87.4, where p is cut off (at -30 p
// is still 9.4e-14 and the slope -29 p); for gelu, whose logistic has 2 sqrt(2/pi)
// (1 + 0.044715 g^2) g for its argument (-1974 at -30), beyond 30, before g^2 grows.
template <int ACT>
__device__ __forceinline__ void gate_slope(float g, float& a, float& s) {
    constexpr float CUT = ACT == QG_ACT_SILU ? 100.0f : 30.0f;
    const float p = logistic<true>(gate_arg<ACT>(g));
    const float c = fminf(fmaxf(g, -CUT), CUT);
    const float dy = ACT == QG_ACT_SILU ? 1.0f : fmaf(3.0f * 0.0713548162726f, c * c, 1.59576912161f);
    a = g * p;
    s = fmaf(c * p * (1.0f - p), dy, p);
}

// Two values of a 16-bit type in a word, rounded to nearest even.
template <typename T> struct Pack;
template <> struct Pack<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    }
};
template <> struct Pack<__half> {
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
};

} // namespace qg
