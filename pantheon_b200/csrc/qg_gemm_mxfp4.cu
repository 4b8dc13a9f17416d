// qg_gemm_mxfp4.cu -- products of MXFP4 operands (qg_mxfp4.cuh) on the sm_100a
// tensor cores: tcgen05.mma kind::mxf4, one ue8m0 scale per 32 along K.
//
//   C[m,n] = out( sum_k (qa[m,k] 2^ea[m,k/32]) (qb[n,k] 2^eb[n,k/32]) )
//   gated: H[m,n] = out( act(A Wg^T)[m,n] * (A Wu^T)[m,n] )
//
// Three kernels (use_rows, launch_gemm): few rows or few tiles
// (qg_gemm_mxfp4_rows.cu), single CTAs for little work, CTA pairs for the rest.  The arithmetic bounds the last: 2 M N K at
// the fp4 rate; measured 4096x8192x8192 94 us (5.8 PFLOP/s, 0.86 of four times the
// measured bf16 rate), 8192x8192x16384 341-348 us (6.3-6.4 PFLOP/s, 0.93), tensor pipe
// 81-86 % active; back to back under the power cap 110 us.
//
// Single CTAs: one persistent CTA per SM, 704 threads, 128 x 256 accumulator columns
// per tile.  The gated form gives columns 0-127 to Wg and 128-255 to Wu (rows
// [128 nt, 128 nt + 128) of each), so one row's gate and up values lie in the
// same TMEM lane and the epilogue joins them in registers.
//   warp 0       producer: per 256-element K block, TMA loads of the A (128
//                rows) and B (256 rows) code tiles (128-byte swizzle) and bulk
//                copies of their scale atoms (up to 1 KB + 2 KB), 4-stage ring.
//   warp 1       TMEM allocator and MMA issuer: 4 x tcgen05.mma M=128 N=256
//                K=64 per K block.
//   warps 2-5    scale writers, one per TMEM lane quarter: each lane moves its
//                16 bytes of every atom from shared memory to TMEM.  An atom
//                covers 128 K here (two MMAs, told apart by the descriptor's
//                scale id 0 / 2), half the scale traffic of the 16-element
//                format.
//   warps 6-21   epilogue: TMEM lane quarter warp % 4, and a quarter of the
//                columns (64) each, held in registers (80 a thread: fp32 results,
//                whose rows are exchanged in twice the words, spill 12 to 56 bytes):
//                the accumulator is free again after two tcgen05.ld per warp, and
//                rounding, activation and stores run under the next tile's MMAs.
// K needs to be a multiple of 32 only: the last K block loads the scale atoms
// and issues the MMAs that K reaches; TMA fills the codes past K with zeros.
// All barrier waits are bounded (qg_ptx.cuh).
#include "qg_common.cuh"
#include "qg_formats.cuh"
#include "qg_gated.cuh"
#include "qg_launch.cuh"
#include "qg_mxfp4.cuh"
#include "qg_mxfp4_mma.cuh"
#include "qg_rows.cuh"

#include <cuda_bf16.h>
#include <atomic>

namespace qg {
namespace mx {

constexpr int BM = 128;
constexpr int BN = 256;                       // accumulator columns (B rows) per tile
constexpr int BK = 256;                       // fp4 elements per K block = 128 bytes per row
constexpr int BK_BYTES = BK / 2;
constexpr int UMMA_K = 64;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK_BYTES;        // 16 KB
constexpr int B_BYTES = BN * BK_BYTES;        // 32 KB
constexpr int ATOMS = BK / ATOM_K;            // scale atoms per 128 rows and K block
constexpr int SFA_BYTES = ATOMS * ATOM_BYTES;         // 1 KB
constexpr int SFB_BYTES = 2 * ATOMS * ATOM_BYTES;     // 2 KB: two 128-row halves
constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
constexpr int SFA_COLS = ATOMS * 4;                   // TMEM columns: four per atom
constexpr int SF_STAGE_COLS = 32;                     // 8 (A) + 16 (B), in two 16-column stores
constexpr int TMEM_COLS = 512;
static_assert(BN + STAGES * SF_STAGE_COLS <= TMEM_COLS, "TMEM budget");
constexpr int GEMM_THREADS = 704;
constexpr int SF_WARP0 = 2;
constexpr int EPI_WARP0 = 6;
constexpr int EPI_WARPS = 16;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
// Tile order: group_m row-tiles share their B tiles in L2 before the next
// columns; a group's rows of A total about 32 MB (the measured best of the
// NVFP4 product at 8 KB rows).
constexpr uint64_t GROUP_A_BYTES = 32ull << 20;

struct Barriers {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t sf_ready[STAGES];
    uint64_t tmem_full;
    uint64_t tmem_empty;
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

constexpr uint32_t SITE_PRODUCER = 0x00060001u;
constexpr uint32_t SITE_MMA_FULL = 0x00060002u;
constexpr uint32_t SITE_MMA_TMEM = 0x00060003u;
constexpr uint32_t SITE_EPI = 0x00060004u;
constexpr uint32_t SITE_SF = 0x00060005u;
constexpr uint32_t SITE_MMA_SF = 0x00060006u;

struct GemmParams {
    int M, N, K;              // gated: N output columns (rows of Wg and of Wu)
    const uint8_t* sfa;
    const uint8_t* sfb;       // B, or Wg
    const uint8_t* sfb2;      // Wu
    void* C;
    uint8_t* SFC;             // scale atoms of an MXFP4 result
    DeviceStatus* status;
    int group_m;
    bool vec;                 // rows of C start on 16 bytes
};

__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int group_m, int& mt, int& nt) {
    const int group = group_m * tiles_n;
    const int g = t / group;
    const int first_m = g * group_m;
    const int gm = min(tiles_m - first_m, group_m);
    const int r = t - g * group;
    mt = first_m + r % gm;
    nt = r / gm;
}

// 32 values of each of the warp's rows row0 + lane, from column n0 on.
template <int OUT>
__device__ __forceinline__ void store32(const GemmParams& p, int row0, int n0, const float (&f)[32]) {
    if (row0 >= p.M || n0 >= p.N) return;
    if constexpr (OUT == QG_OUT_F32) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                              __float_as_uint(f[4 * i + 3]));
        store_rows(static_cast<uint32_t*>(p.C), row0, p.M, n0, p.N, p.vec, v);
    } else {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        store_rows(static_cast<uint16_t*>(p.C), row0, p.M, n0, p.N, p.vec, v);
    }
}

// One K block's scales of a TMEM lane quarter, shared memory -> TMEM columns from
// `col` on, complete before the warp goes on.
__device__ __forceinline__ void move_scales(const uint8_t* sSFA, const uint8_t* sSFB, uint32_t col, int lane) {
    // lane i takes bytes [16 i, 16 i + 16) of each atom.  Columns: A's atoms
    // 0-3 and 4-7, then per atom of K the two halves of B (8 columns).  An atom
    // past K holds what the stage held before; no MMA reads it.
    const uint4* sfa = reinterpret_cast<const uint4*>(sSFA) + lane;
    const uint4* sfb = reinterpret_cast<const uint4*>(sSFB) + lane;
    uint32_t v0[16], v1[16];
    const uint4 a0 = sfa[0], a1 = sfa[32], b00 = sfb[0], b10 = sfb[32], b01 = sfb[64], b11 = sfb[96];
    v0[0] = a0.x; v0[1] = a0.y; v0[2] = a0.z; v0[3] = a0.w;
    v0[4] = a1.x; v0[5] = a1.y; v0[6] = a1.z; v0[7] = a1.w;
    v0[8] = b00.x; v0[9] = b00.y; v0[10] = b00.z; v0[11] = b00.w;
    v0[12] = b01.x; v0[13] = b01.y; v0[14] = b01.z; v0[15] = b01.w;
    v1[0] = b10.x; v1[1] = b10.y; v1[2] = b10.z; v1[3] = b10.w;
    v1[4] = b11.x; v1[5] = b11.y; v1[6] = b11.z; v1[7] = b11.w;
#pragma unroll
    for (int i = 8; i < 16; ++i) v1[i] = 0;
    tmem_st_32x32b_x16(col, v0);
    tmem_st_32x32b_x16(col + 16, v1);
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
}

// Warps SF_WARP0..: the scales of every K block from shared memory to TMEM.
template <int NSTAGES>
__device__ __forceinline__ void write_scales(uint64_t* full, uint64_t* sf_ready, const uint8_t* sSFA, const uint8_t* sSFB,
                                             uint32_t tmem_base, int tiles, int first, int step, int nk,
                                             volatile int* abort_flag, DeviceStatus* status) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + BN;
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
        for (int kb = 0; kb < nk; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort_flag, status, SITE_SF))) {
                ok = false;
                break;
            }
            move_scales(sSFA + stage * SFA_BYTES, sSFB + stage * SFB_BYTES, t_lane + stage * SF_STAGE_COLS, lane);
            if (lane == 0) mbar_arrive(&sf_ready[stage]);
            if (++stage == NSTAGES) { stage = 0; phase ^= 1u; }
        }
    }
}

// Warps EPI_WARP0..: the accumulators of every tile to the output.  `tile_rows`
// rows per tile, this CTA's from row0 on; `tmem_empty` is a cluster address.
template <int OUT, int ACT>
__device__ __forceinline__ void epilogue(const GemmParams& p, uint64_t* tmem_full, uint32_t tmem_empty, uint32_t tmem_base,
                                         int tile_rows, int row0, int tiles_m, int tiles_n, int first, int step,
                                         volatile int* abort_flag) {
    constexpr bool GATED = ACT >= 0;
    constexpr int TN = GATED ? BN / 2 : BN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = tiles_m * tiles_n;
    const int quarter = warp & 3;
    const int part = (warp - EPI_WARP0) >> 2;             // which quarter of the columns
    // gated: 32 gate columns and the 32 up columns of the same outputs
    const uint32_t c0 = GATED ? part * 32 : part * 64;
    const uint32_t c1 = GATED ? BN / 2 + part * 32 : part * 64 + 32;
    const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const int out_blocks = p.N / BLOCK;                    // MXFP4 result
    const int out_kchunks = (p.N + ATOM_K - 1) / ATOM_K;
    const int out_rows = (p.M + 127) / 128 * 128;
    int iter = 0;
    for (int t = first; t < tiles; t += step, ++iter) {
        int mt, nt;
        tile_coords(t, tiles_m, tiles_n, p.group_m, mt, nt);
        if (!warp_wait(tmem_full, iter & 1, abort_flag, p.status, SITE_EPI)) break;
        tc_fence_after();
        uint32_t r0[32], r1[32];
        __syncwarp();
        tmem_ld_32x32b_x32(t_row + c0, r0);
        tmem_ld_32x32b_x32(t_row + c1, r1);
        tmem_ld_wait_regs(r0);
        tmem_ld_wait_regs(r1);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_relaxed(tmem_empty);     // orders TMEM reads only

        const int m_warp = mt * tile_rows + row0 + quarter * 32;
        const int m = m_warp + lane;
        if constexpr (!GATED) {
            const int n0 = nt * BN + part * 64;
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r0[i]);
            store32<OUT>(p, m_warp, n0, f);
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r1[i]);
            store32<OUT>(p, m_warp, n0 + 32, f);
        } else {
            const int n0 = nt * TN + part * 32;
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i)
                f[i] = gated<ACT, OUT != QG_OUT_F32>(__uint_as_float(r0[i]), __uint_as_float(r1[i]));
            if constexpr (OUT == QG_OUT_MXFP4) {
                // these 32 columns are one block of the result
                const int j = nt * 4 + part;
                uint32_t s = 0;
                if (m < p.M && j < out_blocks) {
                    uint32_t amax = 0;
#pragma unroll
                    for (int i = 0; i < 32; ++i) amax = max(amax, __float_as_uint(f[i]) & 0x7FFFFFFFu);
                    s = scale_byte(amax);
                    const float inv = inv_scale(s == 255 ? 0 : s);
                    uint32_t w[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = f[8 * g + i] * inv;
                        w[g] = s == 255 ? 0u : pack8(v);
                    }
                    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.C) + (size_t)m * (p.N / 2) + n0 / 2) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
                // zero past M and N in the atoms' padding (a pair's odd CTA may lie past that too)
                if (m < out_rows) p.SFC[sf_offset(m, j, out_kchunks)] = (uint8_t)s;
            } else {
                store32<OUT>(p, m_warp, n0, f);
            }
        }
    }
}

template <int OUT, int ACT>   // ACT < 0: the plain product
__global__ void __launch_bounds__(GEMM_THREADS, 1)
gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmB2, GemmParams p) {
    constexpr bool GATED = ACT >= 0;
    constexpr int TN = GATED ? BN / 2 : BN;       // output columns per tile
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t* sA = smem;
    uint8_t* sB = sA + STAGES * A_BYTES;
    uint8_t* sSFA = sB + STAGES * B_BYTES;
    uint8_t* sSFB = sSFA + STAGES * SFA_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + STAGES * STAGE_BYTES);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int tiles_m = (p.M + BM - 1) / BM;
    const int tiles_n = (p.N + TN - 1) / TN;
    const int tiles = tiles_m * tiles_n;
    const int nk = (p.K + BK - 1) / BK;
    const int kchunks = (p.K + ATOM_K - 1) / ATOM_K;
    const int b_row_blocks = (p.N + 127) / 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
            mbar_init(&bars->sf_ready[s], 4);
        }
        mbar_init(&bars->tmem_full, 1);
        mbar_init(&bars->tmem_empty, EPI_WARPS);
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        if (GATED) tma_prefetch_desc(&tmB2);
    }
    if (warp == 1) {
        tmem_alloc(&bars->tmem_base, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    volatile int* abort_flag = &bars->abort;
    wait_previous_grid();

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ producer
        uint32_t stage = 0, phase = 0, armed = 0, armed_phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            int mt, nt;
            tile_coords(t, tiles_m, tiles_n, p.group_m, mt, nt);
            for (int kb = 0; kb < nk; ++kb) {
                if (!mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
                const uint32_t atoms = (uint32_t)min(ATOMS, kchunks - kb * ATOMS) * ATOM_BYTES;
                mbar_arrive_expect_tx(&bars->full[stage], A_BYTES + B_BYTES + 3 * atoms);
                tma_load_2d(sA + stage * A_BYTES, &tmA, &bars->full[stage], kb * BK_BYTES, mt * BM);
                bulk_load(sSFA + stage * SFA_BYTES, p.sfa + ((size_t)mt * kchunks + kb * ATOMS) * ATOM_BYTES, atoms,
                          &bars->full[stage]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // a 128-row block past the end of B exists only in a ragged last
                    // tile of the plain product; its columns are never stored, so
                    // block 0's scales stand in for it
                    const int blk = GATED ? nt : nt * 2 + h < b_row_blocks ? nt * 2 + h : 0;
                    const uint8_t* sf = GATED && h ? p.sfb2 : p.sfb;
                    tma_load_2d(sB + stage * B_BYTES + h * (B_BYTES / 2), GATED && h ? &tmB2 : &tmB, &bars->full[stage],
                                kb * BK_BYTES, GATED ? nt * 128 : nt * BN + h * 128);
                    bulk_load(sSFB + stage * SFB_BYTES + h * (SFB_BYTES / 2),
                              sf + ((size_t)blk * kchunks + kb * ATOMS) * ATOM_BYTES, atoms, &bars->full[stage]);
                }
                armed |= 1u << stage;
                armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        // the last releases land before the CTA's shared memory goes away
        for (int i = 0; i < STAGES && ok; ++i) {
            ok = mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER);
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok)
            for (int s = 0; s < STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
    } else if (warp == 1 && lane == 0) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t IDESC0 = idesc_mxf4(BM, BN, 0), IDESC2 = idesc_mxf4(BM, BN, 2);
        uint32_t stage = 0, phase = 0;
        bool ok = true, issued = false;
        int iter = 0;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++iter) {
            if (!mbar_wait(&bars->tmem_empty, (iter & 1) ^ 1u, abort_flag, p.status, SITE_MMA_TMEM)) { ok = false; break; }
            tc_fence_after();
            for (int kb = 0; kb < nk; ++kb) {
                if (!mbar_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_MMA_FULL)) { ok = false; break; }
                if (!mbar_wait(&bars->sf_ready[stage], phase, abort_flag, p.status, SITE_MMA_SF)) { ok = false; break; }
                tc_fence_after();
                const uint32_t sfa_col = tmem_base + BN + stage * SF_STAGE_COLS;
                const uint32_t sfb_col = sfa_col + SFA_COLS;
                const uint32_t a_addr = smem_u32(sA + stage * A_BYTES);
                const uint32_t b_addr = smem_u32(sB + stage * B_BYTES);
                const int steps = min(BK / UMMA_K, (p.K - kb * BK + UMMA_K - 1) / UMMA_K);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)
                    if (k < steps)
                        umma_mxf4(tmem_base, make_sdesc_kmajor_sw128(a_addr + k * (UMMA_K / 2)),
                                  make_sdesc_kmajor_sw128(b_addr + k * (UMMA_K / 2)), (k & 1) ? IDESC2 : IDESC0,
                                  sfa_col + 4 * (k >> 1), sfb_col + 8 * (k >> 1), (kb | k) != 0 ? 1u : 0u);
                issued = true;
                umma_commit(&bars->empty[stage]);
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (ok) umma_commit(&bars->tmem_full);
        }
        if (!ok && issued) {
            umma_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, nullptr, nullptr, 0);
        }
    } else if (warp >= SF_WARP0 && warp < EPI_WARP0) {
        write_scales<STAGES>(bars->full, bars->sf_ready, sSFA, sSFB, tmem_base, tiles, blockIdx.x, gridDim.x, nk, abort_flag,
                             p.status);
    } else if (warp >= EPI_WARP0) {
        epilogue<OUT, ACT>(p, &bars->tmem_full, mapa_shared(smem_u32(&bars->tmem_empty), 0), tmem_base, BM, 0, tiles_m,
                           tiles_n, blockIdx.x, gridDim.x, abort_flag);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
        if (lane == 0 && *abort_flag) atomicAdd(&p.status->drained, 1u);
    }
}

// ---------------------------------------------------------------------------
// CTA pairs: a cluster of two CTAs computes 256 x 256 accumulators
// with tcgen05.mma.cta_group::2 (M = 256, N = 256, K = 64) issued by the even
// CTA.  Per K block a CTA loads its 128 rows of A and 128 of B's 256 rows, 32 KB
// instead of the single CTA's 48 KB, and its tensor core reads 8 KB instead of
// 12 KB of shared memory per MMA: both streams share the 128 bytes per clock of
// shared memory, which is what bounds the single-CTA kernel.  The scales do not
// halve: each CTA's TMEM holds those of its own rows of A and of all 256 rows of
// B.  Protocol beyond the single CTA's:
//   * codes of both CTAs complete on the even CTA's `full` barrier;
//   * a stage is 512 K (two boxes per operand): the MMA thread's waits cost it
//     about 350 clocks a stage, against 1024 clocks of MMAs here and 512 with
//     256 K per stage (111 us at 4096x8192x8192);
//   * scales have rings of their own, in shared memory (filled ahead of the codes by
//     warp 22, freed by the writers) and in TMEM (freed by a commit of the MMAs that
//     read it), so neither a load nor the writers' round trip lies between a freed
//     code stage and its MMAs;
//   * the writers of both CTAs arrive on the even CTA's `sc_ready`, relaxed: what
//     they hand over is in TMEM, complete after tcgen05.wait::st and ordered by the
//     tcgen05 fences on both sides, and a cluster-scope release, which waits for
//     every access of its thread, took 1400 clocks per K block (157 us in all at
//     4096x8192x8192);
//   * the MMA warp commits to the barriers of both CTAs at once; one elected lane of
//     the converged warp issues (a lone lane 0 cost 20 %: 147 us against 117).
constexpr int P_KB = 2;                                        // 256-element K blocks per stage
constexpr int P_STAGES = 3;                                    // code ring
constexpr int P_BLOCK_BYTES = 128 * BK_BYTES;                  // 16 KB: a K block of either operand of a CTA
constexpr int P_OP_BYTES = P_KB * P_BLOCK_BYTES;
constexpr int P_SF_STAGES = 4;                                 // scale ring in shared memory
constexpr int P_SFA_BYTES = P_KB * SFA_BYTES, P_SFB_BYTES = P_KB * SFB_BYTES;
constexpr int P_SF_BYTES = P_SFA_BYTES + P_SFB_BYTES;          // 6 KB
constexpr int P_SF_COLS = P_SF_BYTES / 128;                    // 48 TMEM columns: A's four atoms, then B's per 128 K
constexpr int P_SF_SLOTS = (TMEM_COLS - BN) / P_SF_COLS;       // 5: the scale ring in TMEM
constexpr int P_SMEM_BYTES = P_STAGES * 2 * P_OP_BYTES + P_SF_STAGES * P_SF_BYTES + 1024 + 512;
constexpr int P_THREADS = GEMM_THREADS + 32;
constexpr int SF_LOAD_WARP = EPI_WARP0 + EPI_WARPS;            // 22

struct PairBarriers {
    uint64_t full[P_STAGES];
    uint64_t empty[P_STAGES];
    uint64_t sf_full[P_SF_STAGES];
    uint64_t sf_empty[P_SF_STAGES];
    uint64_t sc_empty[P_SF_SLOTS];   // TMEM scale columns read
    uint64_t sc_ready[P_SF_SLOTS];   // scales in TMEM: the writers of both CTAs (even CTA's only)
    uint64_t tmem_full;
    uint64_t tmem_empty;
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(PairBarriers) <= 512, "barrier block");

__device__ __forceinline__ void umma_mxf4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
        : "memory");
}

template <int OUT, int ACT>
__global__ void __launch_bounds__(P_THREADS, 1)
gemm_mxfp4_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmB2, GemmParams p) {
    constexpr bool GATED = ACT >= 0;
    constexpr int TN = GATED ? BN / 2 : BN;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t* sA = smem;
    uint8_t* sB = sA + P_STAGES * P_OP_BYTES;
    uint8_t* sSFA = sB + P_STAGES * P_OP_BYTES;
    uint8_t* sSFB = sSFA + P_SF_STAGES * P_SFA_BYTES;
    PairBarriers* bars = reinterpret_cast<PairBarriers*>(sSFB + P_SF_STAGES * P_SFB_BYTES);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);   // uniform, and known to be
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int tiles_m = (p.M + 2 * BM - 1) / (2 * BM);
    const int tiles_n = (p.N + TN - 1) / TN;
    const int tiles = tiles_m * tiles_n;
    const int nk = (p.K + BK - 1) / BK;
    const int ns = (nk + P_KB - 1) / P_KB;
    const int kchunks = (p.K + ATOM_K - 1) / ATOM_K;
    const int a_row_blocks = (p.M + 127) / 128, b_row_blocks = (p.N + 127) / 128;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < P_STAGES; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int s = 0; s < P_SF_SLOTS; ++s) {
            mbar_init(&bars->sc_empty[s], 1);
            mbar_init(&bars->sc_ready[s], 8);
        }
        for (int s = 0; s < P_SF_STAGES; ++s) {
            mbar_init(&bars->sf_full[s], 1);
            mbar_init(&bars->sf_empty[s], 4);
        }
        mbar_init(&bars->tmem_full, 1);
        mbar_init(&bars->tmem_empty, 2 * EPI_WARPS);
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        if (GATED) tma_prefetch_desc(&tmB2);
    }
    if (warp == 1) {
        tmem_alloc_pair(&bars->tmem_base, TMEM_COLS);
        tmem_relinquish_pair();
    }
    // both CTAs' barriers initialised and TMEM allocated before anyone signals the other
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    volatile int* abort_flag = &bars->abort;
    wait_previous_grid();

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ code producer (both CTAs)
        uint32_t stage = 0, phase = 0, armed = 0, armed_phase = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs) {
            int mt, nt;
            tile_coords(t, tiles_m, tiles_n, p.group_m, mt, nt);
            const CUtensorMap* b = GATED && !leader ? &tmB2 : &tmB;
            const int b_row = GATED ? nt * 128 : nt * BN + (int)rank * 128;
            for (int kb = 0; kb < nk; kb += P_KB) {
                if (!mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
                const int n = min(P_KB, nk - kb);
                if (leader) mbar_arrive_expect_tx(&bars->full[stage], (uint32_t)n * 4 * P_BLOCK_BYTES);
                const uint32_t full = mapa_shared(smem_u32(&bars->full[stage]), 0);
#pragma unroll
                for (int j = 0; j < P_KB; ++j)
                    if (j < n) {
                        tma_load_2d_pair(sA + stage * P_OP_BYTES + j * P_BLOCK_BYTES, &tmA, full, (kb + j) * BK_BYTES,
                                         mt * 2 * BM + (int)rank * BM);
                        tma_load_2d_pair(sB + stage * P_OP_BYTES + j * P_BLOCK_BYTES, b, full, (kb + j) * BK_BYTES, b_row);
                    }
                armed |= 1u << stage;
                armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == P_STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        // the even CTA's last commits land here before this CTA's shared memory goes away
        for (int i = 0; i < P_STAGES && ok; ++i) {
            ok = mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER);
            if (++stage == P_STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok && leader) {
            // copies of both CTAs complete on the even CTA's barriers: let them land
            for (int s = 0; s < P_STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
        }
    } else if (warp == SF_LOAD_WARP && lane == 0) {
        // ------------------------------------------------------------ scale producer (both CTAs)
        uint32_t stage = 0, phase = 0, armed = 0, armed_phase = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs) {
            int mt, nt;
            tile_coords(t, tiles_m, tiles_n, p.group_m, mt, nt);
            // (128-row blocks past the end of A or B exist only in ragged last tiles; their
            // rows and columns are never stored, so block 0's scales stand in for them)
            const int a_blk = mt * 2 + (int)rank < a_row_blocks ? mt * 2 + (int)rank : 0;
            const uint8_t* sfa = p.sfa + (size_t)a_blk * kchunks * ATOM_BYTES;
            const uint8_t* sfb0 = p.sfb + (size_t)(GATED ? nt : nt * 2) * kchunks * ATOM_BYTES;
            const uint8_t* sfb1 = GATED ? p.sfb2 + (size_t)nt * kchunks * ATOM_BYTES
                                        : p.sfb + (size_t)(nt * 2 + 1 < b_row_blocks ? nt * 2 + 1 : 0) * kchunks * ATOM_BYTES;
            for (int sb = 0; sb < ns; ++sb) {
                if (!mbar_wait(&bars->sf_empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
                const uint32_t atoms = (uint32_t)min(P_KB * ATOMS, kchunks - sb * P_KB * ATOMS) * ATOM_BYTES;
                const size_t at = (size_t)sb * P_KB * ATOMS * ATOM_BYTES;
                uint64_t* full = &bars->sf_full[stage];
                mbar_arrive_expect_tx(full, 3 * atoms);
                bulk_load(sSFA + stage * P_SFA_BYTES, sfa + at, atoms, full);
                bulk_load(sSFB + stage * P_SFB_BYTES, sfb0 + at, atoms, full);
                bulk_load(sSFB + stage * P_SFB_BYTES + P_SFB_BYTES / 2, sfb1 + at, atoms, full);
                armed |= 1u << stage;
                armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == P_SF_STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        if (!ok)
            for (int s = 0; s < P_SF_STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->sf_full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
    } else if (warp == 1 && leader) {
        // ------------------------------------------------------------ MMA issuer (even CTA)
        // The whole warp walks the K blocks and one elected lane issues: descriptors
        // and barrier addresses stay in uniform registers.
        constexpr uint32_t IDESC0 = idesc_mxf4(2 * BM, BN, 0), IDESC2 = idesc_mxf4(2 * BM, BN, 2);
        const uint64_t a_desc0 = make_sdesc_kmajor_sw128(smem_u32(sA)), b_desc0 = make_sdesc_kmajor_sw128(smem_u32(sB));
        uint32_t stage = 0, phase = 0, slot = 0, slot_phase = 0;
        bool ok = true, issued = false;
        int iter = 0;
        for (int t = pair; t < tiles && ok; t += pairs, ++iter) {
            if (!warp_wait(&bars->tmem_empty, (iter & 1) ^ 1u, abort_flag, p.status, SITE_MMA_TMEM)) { ok = false; break; }
            for (int sb = 0; sb < ns; ++sb) {
                if (!warp_wait(&bars->sc_ready[slot], slot_phase, abort_flag, p.status, SITE_MMA_SF) ||
                    !warp_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_MMA_FULL)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sfa_col = tmem_base + BN + slot * P_SF_COLS, sfb_col = sfa_col + P_KB * 8;
                    const uint64_t ad = a_desc0 + stage * (P_OP_BYTES >> 4), bd = b_desc0 + stage * (P_OP_BYTES >> 4);
                    const int steps = (p.K - sb * P_KB * BK + UMMA_K - 1) / UMMA_K;      // all 8 but for the last stage
#pragma unroll
                    for (int k = 0; k < P_KB * BK / UMMA_K; ++k)
                        if (k < steps) {
                            const uint64_t at = (uint64_t)((k / 4) * (P_BLOCK_BYTES >> 4) + (k % 4) * (UMMA_K / 2 >> 4));
                            umma_mxf4_pair(tmem_base, ad + at, bd + at, (k & 1) ? IDESC2 : IDESC0, sfa_col + 4 * (k >> 1),
                                           sfb_col + 8 * (k >> 1), (sb | k) != 0 ? 1u : 0u);
                        }
                    umma_commit_both(&bars->empty[stage]);
                    umma_commit_both(&bars->sc_empty[slot]);
                    if (sb + 1 == ns) umma_commit_both(&bars->tmem_full);
                }
                __syncwarp();
                issued = true;
                if (++stage == P_STAGES) { stage = 0; phase ^= 1u; }
                if (++slot == P_SF_SLOTS) { slot = 0; slot_phase ^= 1u; }
            }
        }
        if (!ok && issued && elect_one()) {
            umma_commit_pair(mapa_shared(smem_u32(&bars->drain), 0));
            mbar_wait(&bars->drain, 0, nullptr, nullptr, 0);
        }
    } else if (warp >= SF_WARP0 && warp < EPI_WARP0) {
        // ------------------------------------------------------------ scale writers (both CTAs)
        const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + BN;
        const int64_t blocks = pair < tiles ? (int64_t)((tiles - pair + pairs - 1) / pairs) * ns : 0;
        uint32_t stage = 0, phase = 0, slot = 0, slot_phase = 0;
        bool ok = true;
        for (int64_t i = 0; i < blocks; ++i) {
            // the scales have landed, and the MMAs that read these TMEM columns are done
            if (!warp_wait(&bars->sf_full[stage], phase, abort_flag, p.status, SITE_SF) ||
                !warp_wait(&bars->sc_empty[slot], slot_phase ^ 1u, abort_flag, p.status, SITE_SF)) {
                ok = false;
                break;
            }
            tc_fence_after();
            // lane i takes bytes [16 i, 16 i + 16) of each atom: four columns.  Atoms past K
            // hold what the stage held before; no MMA reads them.
            const uint4* sfa = reinterpret_cast<const uint4*>(sSFA + stage * P_SFA_BYTES) + lane;
            const uint4* sfb = reinterpret_cast<const uint4*>(sSFB + stage * P_SFB_BYTES) + lane;
            uint32_t va[16], vb[16], vc[16];
#pragma unroll
            for (int k = 0; k < P_KB * ATOMS; ++k) {
                const uint4 x = sfa[k * 32], y = sfb[k * 32], z = sfb[(P_KB * ATOMS + k) * 32];
                uint32_t* d = k < 2 ? vb + 8 * k : vc + 8 * (k - 2);
                va[4 * k] = x.x; va[4 * k + 1] = x.y; va[4 * k + 2] = x.z; va[4 * k + 3] = x.w;
                d[0] = y.x; d[1] = y.y; d[2] = y.z; d[3] = y.w;
                d[4] = z.x; d[5] = z.y; d[6] = z.z; d[7] = z.w;
            }
            const uint32_t col = t_lane + slot * P_SF_COLS;
            tmem_st_32x32b_x16(col, va);
            tmem_st_32x32b_x16(col + 16, vb);
            tmem_st_32x32b_x16(col + 32, vc);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_relaxed(mapa_shared(smem_u32(&bars->sc_ready[slot]), 0));
                mbar_arrive(&bars->sf_empty[stage]);
            }
            if (++stage == P_SF_STAGES) { stage = 0; phase ^= 1u; }
            if (++slot == P_SF_SLOTS) { slot = 0; slot_phase ^= 1u; }
        }
        for (int i = 0; i < P_SF_SLOTS && ok; ++i) {          // (as the code producer: the last commits)
            ok = warp_wait(&bars->sc_empty[slot], slot_phase ^ 1u, abort_flag, p.status, SITE_SF);
            if (++slot == P_SF_SLOTS) { slot = 0; slot_phase ^= 1u; }
        }
    } else if (warp >= EPI_WARP0 && warp < EPI_WARP0 + EPI_WARPS) {
        epilogue<OUT, ACT>(p, &bars->tmem_full, mapa_shared(smem_u32(&bars->tmem_empty), 0), tmem_base, 2 * BM,
                           (int)rank * BM, tiles_m, tiles_n, pair, pairs, abort_flag);
    }

    // the even CTA's MMAs read this CTA's shared memory and write its TMEM:
    // neither CTA frees anything before both are done
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
        if (lane == 0 && *abort_flag) atomicAdd(&p.status->drained, 1u);
    }
}

// CTA pairs that can be resident at once (a pair needs two free SMs of one GPC,
// so this can be below half of the SMs).  All variants have the same block and
// shared-memory size.
static int resident_pairs(int* out, const DeviceInfo* info) {
    static std::atomic<int> resident[64];                      // 0: not asked yet
    int dev = 0;
    QG_CUDA(cudaGetDevice(&dev));
    if (!resident[dev & 63]) {
        cudaLaunchConfig_t lc = {};
        lc.gridDim = dim3(info->sm_count & ~1);
        lc.blockDim = dim3(P_THREADS);
        lc.dynamicSmemBytes = P_SMEM_BYTES;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {2, 1, 1};
        lc.attrs = at;
        lc.numAttrs = 1;
        int n = 0;
        auto kernel = gemm_mxfp4_pair_kernel<QG_OUT_BF16, -1>;
        QG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM_BYTES));
        QG_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &lc));
        resident[dev & 63] = n > 0 ? n : 1;
    }
    *out = resident[dev & 63];
    return QG_OK;
}

template <int OUT, int ACT>
static int launch_gemm(const void* A, const void* B, const void* B2, GemmParams p, cudaStream_t stream) {
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
    if (use_rows(p.M, p.N, p.K, ACT >= 0, info->sm_count))
        return gemm_rows(A, p.sfa, B, p.sfb, B2, p.sfb2, p.C, p.SFC, OUT, ACT, p.vec, p.M, p.N, p.K, info->sm_count, stream);
    if ((rc = device_status_ptr(&p.status))) return rc;
    CUtensorMap tmA, tmB, tmB2;
    const uint64_t row = (uint64_t)p.K / 2;
    if ((rc = make_tmap_2d(&tmA, A, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, (uint64_t)p.M, row, BK_BYTES, BM,
                           CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    if ((rc = make_tmap_2d(&tmB, B, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, (uint64_t)p.N, row, BK_BYTES, 128,
                           CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    tmB2 = tmB;
    if (ACT >= 0 && (rc = make_tmap_2d(&tmB2, B2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, (uint64_t)p.N, row, BK_BYTES,
                                       128, CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    const uint64_t group = GROUP_A_BYTES / ((uint64_t)BM * row);
    p.group_m = (int)(group < 1 ? 1 : group > 64 ? 64 : group);
    const int tiles_n = ceil_div(p.N, ACT >= 0 ? BN / 2 : BN);
    // Pairs above 128 rows, unless one wave of single CTAs does it with a short K, where
    // a pair's longer start shows (us, single / pairs: 160x4096x1024 5.6 / 6.5,
    // 512x8192x2048 7.7 / 8.7, 1024x4096x4096 10.8 / 11.2, 512x4096x4096 10.4 / 10.1,
    // 512x8192x8192 18.0 / 16.6).
    const int64_t singles = (int64_t)ceil_div(p.M, BM) * tiles_n;
    if (p.M > BM && (singles > info->sm_count || p.K > 16 * BK)) {
        QG_CUDA(cudaFuncSetAttribute(gemm_mxfp4_pair_kernel<OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     P_SMEM_BYTES));
        int pairs = 0;
        if ((rc = resident_pairs(&pairs, info))) return rc;
        p.group_m = p.group_m > 1 ? p.group_m / 2 : 1;             // in 256-row tiles
        const int64_t tiles = (int64_t)ceil_div(p.M, 2 * BM) * tiles_n;
        if (tiles < pairs) pairs = (int)tiles;
        QG_CUDA(launch_overlapped(gemm_mxfp4_pair_kernel<OUT, ACT>, dim3(2 * pairs), dim3(P_THREADS), P_SMEM_BYTES,
                                  stream, 2, tmA, tmB, tmB2, p));
        return QG_OK;
    }
    QG_CUDA(cudaFuncSetAttribute(gemm_mxfp4_kernel<OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    const int grid = singles < info->sm_count ? (int)singles : info->sm_count;
    QG_CUDA(launch_overlapped(gemm_mxfp4_kernel<OUT, ACT>, dim3(grid), dim3(GEMM_THREADS), SMEM_BYTES, stream, 1, tmA, tmB,
                              tmB2, p));
    return QG_OK;
}

static int check_mx(const char* name, const void* A, const void* SFA, const void* B, const void* SFB, const void* C,
                    int M, int N, int K) {
    QG_CHECK_ARG(A && SFA && B && SFB && C, "%s: null operand or output", name);
    QG_CHECK_ARG(M > 0 && N > 0 && K > 0, "%s: empty shape %dx%dx%d", name, M, N, K);
    QG_CHECK_ARG(K % 32 == 0, "%s: K=%d must be a multiple of 32", name, K);
    QG_CHECK_ARG(M <= (1 << 30) && N <= (1 << 30) && K <= (1 << 30) &&
                     (int64_t)ceil_div(M, BM) * ceil_div(N, BN / 2) <= (1 << 30),
                 "%s: shape %dx%dx%d is too large", name, M, N, K);
    QG_CHECK_ARG((((uintptr_t)A | (uintptr_t)SFA | (uintptr_t)B | (uintptr_t)SFB) & 15) == 0,
                 "%s: codes and scales must be 16-byte aligned", name);
    return QG_OK;
}

} // namespace mx

int gemm_mxfp4(const void* A, const void* SFA, const void* B, const void* SFB, void* C, int out_type, int M, int N,
               int K, cudaStream_t stream) {
    int rc = mx::check_mx("qg_gemm_mxfp4", A, SFA, B, SFB, C, M, N, K);
    if (rc) return rc;
    mx::GemmParams p{M, N, K, static_cast<const uint8_t*>(SFA), static_cast<const uint8_t*>(SFB), nullptr, C, nullptr,
                     nullptr, 1, false};
    switch (out_type) {
        case QG_OUT_BF16:
            QG_CHECK_ARG((uintptr_t)C % 2 == 0, "qg_gemm_mxfp4: C is not aligned to its element");
            p.vec = N % 8 == 0 && ((uintptr_t)C & 15) == 0;
            return mx::launch_gemm<QG_OUT_BF16, -1>(A, B, nullptr, p, stream);
        case QG_OUT_F32:
            QG_CHECK_ARG((uintptr_t)C % 4 == 0, "qg_gemm_mxfp4: C is not aligned to its element");
            p.vec = N % 4 == 0 && ((uintptr_t)C & 15) == 0;
            return mx::launch_gemm<QG_OUT_F32, -1>(A, B, nullptr, p, stream);
        default: set_error("qg_gemm_mxfp4: out_type %d (bf16 or f32)", out_type); return QG_ERR_ARG;
    }
}

int gemm_gated_mxfp4(const void* A, const void* SFA, const void* Wg, const void* SFG, const void* Wu, const void* SFU,
                     void* H, void* SFH, int out_type, int act, int M, int N, int K, cudaStream_t stream) {
    int rc = mx::check_mx("qg_gemm_gated_mxfp4", A, SFA, Wg, SFG, H, M, N, K);
    if (rc) return rc;
    QG_CHECK_ARG(Wu && SFU, "qg_gemm_gated_mxfp4: null operand or output");
    QG_CHECK_ARG((((uintptr_t)Wu | (uintptr_t)SFU) & 15) == 0, "qg_gemm_gated_mxfp4: codes and scales must be 16-byte aligned");
    QG_CHECK_ARG(act == QG_ACT_SILU || act == QG_ACT_GELU_TANH, "qg_gemm_gated_mxfp4: unknown activation %d", act);
    mx::GemmParams p{M, N, K, static_cast<const uint8_t*>(SFA), static_cast<const uint8_t*>(SFG),
                     static_cast<const uint8_t*>(SFU), H, static_cast<uint8_t*>(SFH), nullptr, 1, false};
    const bool silu = act == QG_ACT_SILU;
    switch (out_type) {
        case QG_OUT_BF16:
            QG_CHECK_ARG((uintptr_t)H % 2 == 0, "qg_gemm_gated_mxfp4: H is not aligned to its element");
            p.vec = N % 8 == 0 && ((uintptr_t)H & 15) == 0;
            return silu ? mx::launch_gemm<QG_OUT_BF16, QG_ACT_SILU>(A, Wg, Wu, p, stream)
                        : mx::launch_gemm<QG_OUT_BF16, QG_ACT_GELU_TANH>(A, Wg, Wu, p, stream);
        case QG_OUT_F32:
            QG_CHECK_ARG((uintptr_t)H % 4 == 0, "qg_gemm_gated_mxfp4: H is not aligned to its element");
            p.vec = N % 4 == 0 && ((uintptr_t)H & 15) == 0;
            return silu ? mx::launch_gemm<QG_OUT_F32, QG_ACT_SILU>(A, Wg, Wu, p, stream)
                        : mx::launch_gemm<QG_OUT_F32, QG_ACT_GELU_TANH>(A, Wg, Wu, p, stream);
        case QG_OUT_MXFP4:
            QG_CHECK_ARG(SFH, "qg_gemm_gated_mxfp4: an MXFP4 result needs its scale buffer");
            QG_CHECK_ARG(N % 32 == 0, "qg_gemm_gated_mxfp4: N=%d must be a multiple of 32 for an MXFP4 result", N);
            QG_CHECK_ARG((((uintptr_t)H | (uintptr_t)SFH) & 15) == 0,
                         "qg_gemm_gated_mxfp4: an MXFP4 result must be 16-byte aligned");
            return silu ? mx::launch_gemm<QG_OUT_MXFP4, QG_ACT_SILU>(A, Wg, Wu, p, stream)
                        : mx::launch_gemm<QG_OUT_MXFP4, QG_ACT_GELU_TANH>(A, Wg, Wu, p, stream);
        default: set_error("qg_gemm_gated_mxfp4: out_type %d (bf16, f32 or mxfp4)", out_type); return QG_ERR_ARG;
    }
}

} // namespace qg

extern "C" int qg_gemm_mxfp4(const void* A, const void* SFA, const void* B, const void* SFB, void* C, int out_type,
                             int M, int N, int K, void* stream) {
    return qg::gemm_mxfp4(A, SFA, B, SFB, C, out_type, M, N, K, static_cast<cudaStream_t>(stream));
}

extern "C" int qg_gemm_gated_mxfp4(const void* A, const void* SFA, const void* Wg, const void* SFG, const void* Wu,
                                   const void* SFU, void* H, void* SFH, int out_type, int act, int M, int N, int K,
                                   void* stream) {
    return qg::gemm_gated_mxfp4(A, SFA, Wg, SFG, Wu, SFU, H, SFH, out_type, act, M, N, K,
                                static_cast<cudaStream_t>(stream));
}
