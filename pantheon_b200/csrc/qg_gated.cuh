// qg_gated.cuh -- the activations of the gated products, and their slopes.
//
//   silu(g)      = g / (1 + exp(-g))
//   gelu_tanh(g) = 0.5 g (1 + tanh(z)) = g / (1 + exp(-2 z)),  z = sqrt(2/pi) (g + 0.044715 g^3)
// (0.5 (1 + tanh z) is the logistic function of 2 z), so both are g p with
// p = 1 / (1 + exp(-y)), and their slopes are p + g p (1 - p) dy/dg.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/pantheon_qgemm.h"

namespace qg {

// The logistic's argument of activation ACT.
template <int ACT>
__device__ __forceinline__ float gate_arg(float g) {
    if constexpr (ACT == QG_ACT_SILU) return g;
    else return g * fmaf(0.0713548162726f, g * g, 1.59576912161f);   // 2 sqrt(2/pi) (1 + 0.044715 g^2) g
}

// FAST: the hardware's 2^x and reciprocal, a few units in the last place of
// fp32, for results that are rounded to 16 bits or fewer.  At y = -88 and below
// exp(-y) passes the largest fp32 and p is 0, its limit.
template <bool FAST>
__device__ __forceinline__ float logistic(float y) {
    if constexpr (FAST) return __fdividef(1.0f, 1.0f + __expf(fminf(-y, 87.0f)));
    else return 1.0f / (1.0f + expf(-y));
}

template <int ACT, bool FAST>
__device__ __forceinline__ float gated(float g, float u) {
    return g * logistic<FAST>(gate_arg<ACT>(g)) * u;
}

} // namespace qg
