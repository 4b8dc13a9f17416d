// qg_few_rows.cuh -- how the kernels for few rows (qg_gemm_mxfp4_rows.cu,
// qg_gemm_gated_rows.cu) cut a product: rows of a tile, and CTAs of a cluster that
// share its contraction.  Host code, without CUDA.  Two of their CTAs fit an SM, so
// `2 * sms` are one wave; `tiles_n` weight tiles of 128 rows (gated: 64 + 64).
// Both kernels' contraction blocks (256 MXFP4 or 64 two-byte elements) have as many
// bytes, so they share the rules; figures below in us.
#pragma once

#include <cstdint>

namespace qg {
namespace few_rows {

inline int64_t tiles_of(int M, int rows) { return ((int64_t)M + rows - 1) / rows; }

// Whether every tile of 64 rows finds four CTAs in one wave.
inline bool few_tiles(int M, int tiles_n, int sms) { return 4 * (int64_t)tiles_n * tiles_of(M, 64) <= 2 * (int64_t)sms; }

// Rows per tile: 128 only where they are many.  128 / 64 rows, MXFP4: 128x1024x4096
// 6.4 / 5.3, 512x1024x8192 10.5 / 8.4; 512x1024x4096 6.8 / 6.9 and 333x1001x4128 7.4 /
// 7.7 lose by it.  bf16 block: 128x1024x1024 6.5 / 5.3, 256x1024x4096 12.5 / 11.0;
// 65x4096x4096 16.3 / 19.3 and 512x1024x4096 14.4 / 15.8 (not few, so 128).
inline int row_tile(int M, int tiles_n, int sms) {
    if (M <= 64) return M <= 16 ? 16 : M <= 32 ? 32 : 64;
    return few_tiles(M, tiles_n, sms) ? 64 : 128;
}

// CTAs that share a tile's contraction of `nk` blocks: as many as one wave holds,
// four blocks each at least.  A CTA's start and end cost 2-3 us, which a second wave
// pays again, and the join grows with the split.  MXFP4, one row, K=8192: N=28672
// 22.8 unsplit, 26.1 in two, 31.5 in four; N=8192 14.1, 10.7, 10.4 and 13.9 in eight;
// N=1024 13.3, 8.6, 6.2, 5.1.  333 x 1001 x 4128 (17 blocks): 7.4 in four, 9.6 in
// eight (tiles of 128 rows).
inline int pick_split(int M, int tiles_n, int nk, int sms) {
    const int64_t tiles = tiles_n * tiles_of(M, row_tile(M, tiles_n, sms));
    int split = 1;
    while (split < 8 && 2 * split * tiles <= 2 * (int64_t)sms && 8 * split <= nk) split *= 2;
    return split;
}

} // namespace few_rows
} // namespace qg
