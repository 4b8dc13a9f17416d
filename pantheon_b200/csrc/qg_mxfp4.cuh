// qg_mxfp4.cuh -- the MXFP4 format (OCP Microscaling v1.0): 32 consecutive
// values along K share one power-of-two scale, stored as the biased exponent
// byte s (ue8m0: 2^(s-127), 255 = NaN); each value is an e2m1 code
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).
//
// Conversion of a block, all exact in fp32 but for the last rounding:
//   e = max(floor(log2(max |x|)) - 2, -127), s = e + 127
//   q = e2m1(x * 2^-e), to the nearest, ties to the even code, |q| <= 6
// (2 is the exponent of e2m1's largest power of two, so a block's maximum lands
// in [4, 8) and saturates at 6).  A block of zeros gets s = 0; a block that
// holds a NaN or an infinity gets s = 255 and codes 0: all of it reads as NaN.
//
// Codes: two per byte along K, low nibble = even k.  Scales: 512-byte atoms of
// 128 rows x 4 blocks (128 K), atoms ordered [row block][K/128]; inside an
// atom row r's four scales are bytes (r%32)*16 + ((r/32)%4)*4 + 0..3, the order
// in which tcgen05.mma reads them from TMEM.  Scale bytes of rows and blocks
// past the tensor are zero (a 255 there would turn the zero codes that pad K
// into NaN).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace qg {
namespace mx {

constexpr int BLOCK = 32;
constexpr int ATOM_BYTES = 512;
constexpr int ATOM_K = 128;

// Byte of row r's scale of block j; `kchunks` = ceil(K / 128).
__device__ __forceinline__ size_t sf_offset(int r, int j, int kchunks) {
    return ((size_t)(r >> 7) * kchunks + (size_t)(j >> 2)) * ATOM_BYTES +
           (size_t)((r & 31) * 16 + ((r >> 5) & 3) * 4 + (j & 3));
}

// Scale byte of a block whose largest magnitude has the fp32 bits `amax`
// (the sign cleared; every NaN compares above infinity as an integer).
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
    const int e = (int)(amax >> 23) - 2;               // floor(log2) - 2 + 127; subnormals give -2
    return amax >= 0x7F800000u ? 255u : (uint32_t)(e > 0 ? e : 0);
}

// 2^(127 - s), the factor that brings a block into the range of e2m1 (s <= 252: normal).
__device__ __forceinline__ float inv_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }

// 2^(s - 127), NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7FFFFFFFu : s << 23);
}

// Eight values to eight codes (value i in nibble i), nearest even, saturating.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    uint32_t w;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}

// Two values to two codes, the first in the low nibble.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t w;
    asm("{\n\t.reg .b8 a;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "mov.b32 %0, {a, a, a, a};\n\t}"
        : "=r"(w) : "f"(lo), "f"(hi));
    return w & 0xFFu;
}

} // namespace mx
} // namespace qg
