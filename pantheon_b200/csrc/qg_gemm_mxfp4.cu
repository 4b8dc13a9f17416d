// qg_gemm_mxfp4.cu -- products of MXFP4 operands (qg_mxfp4.cuh) on the sm_100a
// tensor cores: tcgen05.mma kind::mxf4, one ue8m0 scale per 32 along K.
//
//   C[m,n] = out( sum_k (qa[m,k] 2^ea[m,k/32]) (qb[n,k] 2^eb[n,k/32]) )
//   gated: H[m,n] = out( act(A Wg^T)[m,n] * (A Wu^T)[m,n] )
//
// One persistent CTA per SM, 704 threads, 128 x 256 accumulator columns per
// tile.  The gated form gives columns 0-127 to Wg and 128-255 to Wu (rows
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
//                columns (64) each, which fit in its registers: the accumulator
//                is free again after two tcgen05.ld per warp, and rounding,
//                activation and stores run under the next tile's MMAs.
// K needs to be a multiple of 32 only: the last K block loads the scale atoms
// and issues the MMAs that K reaches; TMA fills the codes past K with zeros.
// All barrier waits are bounded (qg_ptx.cuh).
#include "qg_common.cuh"
#include "qg_formats.cuh"
#include "qg_gated.cuh"
#include "qg_mxfp4.cuh"

#include <cuda_bf16.h>

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

// Store COLS values of one output row from column n0 on (columns past N are left out).
template <int OUT, int COLS>
__device__ __forceinline__ void store_row(void* C, size_t row, int n0, int N, bool vec, const float (&f)[COLS]) {
    if constexpr (OUT == QG_OUT_F32) {
        float* dst = static_cast<float*>(C) + row * N + n0;
        if (vec && n0 + COLS <= N) {
#pragma unroll
            for (int i = 0; i < COLS; i += 4)
                *reinterpret_cast<float4*>(dst + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < COLS; ++i)
                if (n0 + i < N) dst[i] = f[i];
        }
    } else {
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(C) + row * N + n0;
        if (vec && n0 + COLS <= N) {
#pragma unroll
            for (int i = 0; i < COLS; i += 8) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(f[i + 2 * j], f[i + 2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
                *reinterpret_cast<uint4*>(dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < COLS; ++i)
                if (n0 + i < N) dst[i] = __float2bfloat16_rn(f[i]);
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
        // ------------------------------------------------------------ scale writers
        const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + BN;
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            for (int kb = 0; kb < nk; ++kb) {
                if (!__all_sync(0xffffffffu, mbar_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_SF))) {
                    ok = false;
                    break;
                }
                // lane i takes bytes [16 i, 16 i + 16) of each atom.  Columns: A's atoms
                // 0-3 and 4-7, then per atom of K the two halves of B (8 columns).  An atom
                // past K holds what the stage held before; no MMA reads it.
                const uint4* sfa = reinterpret_cast<const uint4*>(sSFA + stage * SFA_BYTES) + lane;
                const uint4* sfb = reinterpret_cast<const uint4*>(sSFB + stage * SFB_BYTES) + lane;
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
                const uint32_t col = t_lane + stage * SF_STAGE_COLS;
                tmem_st_32x32b_x16(col, v0);
                tmem_st_32x32b_x16(col + 16, v1);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->sf_ready[stage]);
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp >= EPI_WARP0) {
        // ------------------------------------------------------------ epilogue
        const int quarter = warp & 3;
        const int part = (warp - EPI_WARP0) >> 2;             // which quarter of the columns
        const int row = quarter * 32 + lane;
        // gated: 32 gate columns and the 32 up columns of the same outputs
        const uint32_t c0 = GATED ? part * 32 : part * 64;
        const uint32_t c1 = GATED ? BN / 2 + part * 32 : part * 64 + 32;
        const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const int out_blocks = p.N / BLOCK;                    // MXFP4 result
        const int out_kchunks = (p.N + ATOM_K - 1) / ATOM_K;
        int iter = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++iter) {
            int mt, nt;
            tile_coords(t, tiles_m, tiles_n, p.group_m, mt, nt);
            int ok = 1;
            if (lane == 0) ok = mbar_wait(&bars->tmem_full, iter & 1, abort_flag, p.status, SITE_EPI) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            tc_fence_after();
            uint32_t r0[32], r1[32];
            __syncwarp();
            tmem_ld_32x32b_x32(t_row + c0, r0);
            tmem_ld_32x32b_x32(t_row + c1, r1);
            tmem_ld_wait_regs(r0);
            tmem_ld_wait_regs(r1);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->tmem_empty);

            const int m = mt * BM + row;
            if constexpr (!GATED) {
                if (m >= p.M) continue;
                const int n0 = nt * BN + part * 64;
                float f[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r0[i]);
                if (n0 < p.N) store_row<OUT, 32>(p.C, m, n0, p.N, p.vec, f);
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r1[i]);
                if (n0 + 32 < p.N) store_row<OUT, 32>(p.C, m, n0 + 32, p.N, p.vec, f);
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
                    p.SFC[sf_offset(m, j, out_kchunks)] = (uint8_t)s;   // zero past M and N: the atoms' padding
                } else {
                    if (m < p.M && n0 < p.N) store_row<OUT, 32>(p.C, m, n0, p.N, p.vec, f);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
        if (lane == 0 && *abort_flag) atomicAdd(&p.status->drained, 1u);
    }
}

template <int OUT, int ACT>
static int launch_gemm(const void* A, const void* B, const void* B2, GemmParams p, cudaStream_t stream) {
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
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
    QG_CUDA(cudaFuncSetAttribute(gemm_mxfp4_kernel<OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    const uint64_t group = GROUP_A_BYTES / ((uint64_t)BM * row);
    p.group_m = (int)(group < 1 ? 1 : group > 64 ? 64 : group);
    const int64_t tiles = (int64_t)ceil_div(p.M, BM) * ceil_div(p.N, ACT >= 0 ? BN / 2 : BN);
    const int grid = tiles < info->sm_count ? (int)tiles : info->sm_count;
    gemm_mxfp4_kernel<OUT, ACT><<<grid, GEMM_THREADS, SMEM_BYTES, stream>>>(tmA, tmB, tmB2, p);
    QG_CUDA(cudaGetLastError());
    return QG_OK;
}

static int check_mx(const char* name, const void* A, const void* SFA, const void* B, const void* SFB, const void* C,
                    int M, int N, int K) {
    QG_CHECK_ARG(A && SFA && B && SFB && C, "%s: null operand or output", name);
    QG_CHECK_ARG(M > 0 && N > 0 && K > 0, "%s: empty shape %dx%dx%d", name, M, N, K);
    QG_CHECK_ARG(K % 32 == 0, "%s: K=%d must be a multiple of 32", name, K);
    QG_CHECK_ARG((int64_t)ceil_div(M, BM) * ceil_div(N, BN / 2) <= INT32_MAX / 2, "%s: shape %dx%d is too large", name, M, N);
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
