// qg_gemm_mxfp4_rows.cu -- the products of qg_gemm_mxfp4.cu for few rows of A
// (decode steps, short prompts; more rows where a long K meets few tiles), where reading the weights once is the whole
// cost: K (1/2 + 1/32) bytes per weight row against NT columns of arithmetic.
//
// The operands change places: a tile takes 128 weight rows as the M side of
// tcgen05.mma (gated: 64 rows of Wg and the same 64 of Wu) and NT = 16, 32, 64
// or 128 rows of A as its N side, so few rows waste no tensor-core rows and the
// accumulator is small.  K is split over the CTAs of a cluster (1 to 8); each
// sums its part in TMEM, puts the partial tile in its shared memory, and every
// CTA of the cluster joins a share of the rows from all of them over
// distributed shared memory, in rank order: no workspace, no atomics, the same
// bits on every run.
//
// Measured: 1x28672x8192 21.9 us (125 MB, 5.7 TB/s, 0.87 of the measured copy
// bandwidth), 1x8192x8192 9.1, 1x1024x8192 3.9; gated 16x14336x4096 13.6 us (0.71).
// What is left above the bytes is a launch's start and end, 3-4 us.
//
// 192 threads, two CTAs per SM:
//   warp 0      producer: code tiles by TMA and scale atoms by bulk copies, per
//               256-element K block, into a ring of up to 105 KB.
//   warp 1      TMEM allocator and MMA issuer.
//   warps 2-5   scale writers (shared memory -> TMEM), then the epilogue.
// All barrier waits are bounded (qg_ptx.cuh).
#include "qg_common.cuh"
#include "qg_few_rows.cuh"
#include "qg_formats.cuh"
#include "qg_gated.cuh"
#include "qg_launch.cuh"
#include "qg_mxfp4.cuh"
#include "qg_mxfp4_mma.cuh"
#include "qg_rows.cuh"

#include <cuda_bf16.h>

namespace qg {
namespace mx {
namespace rows {

constexpr int BW = 128;                        // weight rows of a tile
constexpr int BK = 256;
constexpr int BK_BYTES = BK / 2;
constexpr int UMMA_K = 64;
constexpr int W_BYTES = BW * BK_BYTES;         // 16 KB
constexpr int SF_BYTES = 2 * ATOM_BYTES;       // 1 KB: the atoms of 128 rows and one K block
constexpr int THREADS = 192;
constexpr int SF_COLS = 16;                    // TMEM columns of a stage's scales: 8 weight, 8 A

template <int NT, bool GATED>
struct Cfg {
    static constexpr int X_BYTES = NT * BK_BYTES;
    static constexpr int SFW = (GATED ? 2 : 1) * SF_BYTES;
    static constexpr int STAGE = W_BYTES + X_BYTES + SFW + SF_BYTES;
    static constexpr int STAGES = 105 * 1024 / STAGE;       // two CTAs share an SM's 227 KB
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
    static constexpr int COLS = NT + STAGES * SF_COLS;
    static constexpr int TMEM_COLS = COLS <= 128 ? 128 : 256;
    static_assert(COLS <= 256, "two CTAs share TMEM");
    static_assert(NT * BW * 4 <= STAGES * STAGE, "the partial tile fits the ring");
};

constexpr uint32_t SITE_PRODUCER = 0x00080001u;
constexpr uint32_t SITE_MMA_FULL = 0x00080002u;
constexpr uint32_t SITE_MMA_SF = 0x00080003u;
constexpr uint32_t SITE_EPI = 0x00080004u;
constexpr uint32_t SITE_SF = 0x00080005u;

struct Params {
    int M, N, K;
    const uint8_t* sfx;       // A's scales
    const uint8_t* sfw;       // B's, or Wg's
    const uint8_t* sfw2;      // Wu's
    void* C;
    uint8_t* SFC;
    DeviceStatus* status;
    bool vec;
};

template <int MAX>
struct Barriers {
    uint64_t full[MAX];
    uint64_t empty[MAX];
    uint64_t sf_ready[MAX];
    uint64_t acc_full;
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

template <int NT, int OUT, int ACT>   // ACT < 0: the plain product
__global__ void __launch_bounds__(THREADS, 2)
rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
            const __grid_constant__ CUtensorMap tmW2, Params p) {
    constexpr bool GATED = ACT >= 0;
    using G = Cfg<NT, GATED>;
    constexpr int TN = GATED ? BW / 2 : BW;          // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t* sW = smem;
    uint8_t* sX = sW + G::STAGES * W_BYTES;
    uint8_t* sSFW = sX + G::STAGES * G::X_BYTES;
    uint8_t* sSFX = sSFW + G::STAGES * G::SFW;
    using Bars = Barriers<G::STAGES>;
    static_assert(sizeof(Bars) <= 256, "barrier block");
    Bars* bars = reinterpret_cast<Bars*>(smem + G::STAGES * G::STAGE);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const int wt = blockIdx.x / ranks;               // weight tile
    const int m0 = blockIdx.y * NT;
    const int nk_all = (p.K + BK - 1) / BK;
    const int kb0 = (int)((int64_t)nk_all * rank / ranks), kb1 = (int)((int64_t)nk_all * (rank + 1) / ranks);
    const int kchunks = (p.K + ATOM_K - 1) / ATOM_K;

    if (threadIdx.x == 0) {
        for (int s = 0; s < G::STAGES; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
            mbar_init(&bars->sf_ready[s], 4);
        }
        mbar_init(&bars->acc_full, 1);
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&bars->tmem_base, G::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    volatile int* abort_flag = &bars->abort;
    wait_previous_grid();
    float* part = reinterpret_cast<float*>(smem);    // [row of A][128 weight rows], over the ring once it is drained

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ producer
        uint32_t stage = 0, phase = 0, armed = 0, armed_phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
            uint64_t* full = &bars->full[stage];
            const uint32_t atoms = (uint32_t)min(2, kchunks - kb * 2) * ATOM_BYTES;
            mbar_arrive_expect_tx(full, W_BYTES + G::X_BYTES + (GATED ? 3 : 2) * atoms);
            const size_t sf_at = (size_t)kb * 2 * ATOM_BYTES;
            const size_t sf_row = (size_t)kchunks * ATOM_BYTES;      // atoms of a 128-row block
            uint8_t* w = sW + stage * W_BYTES;
            uint8_t* sw = sSFW + stage * G::SFW;
            tma_load_2d(w, &tmW, full, kb * BK_BYTES, wt * TN);
            if (GATED) {
                tma_load_2d(w + W_BYTES / 2, &tmW2, full, kb * BK_BYTES, wt * TN);
                bulk_load(sw, p.sfw + (wt >> 1) * sf_row + sf_at, atoms, full);
                bulk_load(sw + SF_BYTES, p.sfw2 + (wt >> 1) * sf_row + sf_at, atoms, full);
            } else {
                bulk_load(sw, p.sfw + wt * sf_row + sf_at, atoms, full);
            }
            tma_load_2d(sX + stage * G::X_BYTES, &tmX, full, kb * BK_BYTES, m0);
            bulk_load(sSFX + stage * SF_BYTES, p.sfx + (m0 >> 7) * sf_row + sf_at, atoms, full);
            armed |= 1u << stage;
            armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
            if (++stage == G::STAGES) { stage = 0; phase ^= 1u; }
        }
        // the last releases land before the CTA's shared memory goes away
        for (int i = 0; i < G::STAGES && ok; ++i) {
            ok = mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER);
            if (++stage == G::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok)
            for (int s = 0; s < G::STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
    } else if (warp == 1 && lane == 0) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t IDESC0 = idesc_mxf4(BW, NT, 0), IDESC2 = idesc_mxf4(BW, NT, 2);
        uint32_t stage = 0, phase = 0;
        bool ok = true, issued = false;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_MMA_FULL)) { ok = false; break; }
            if (!mbar_wait(&bars->sf_ready[stage], phase, abort_flag, p.status, SITE_MMA_SF)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sfw_col = tmem_base + NT + stage * SF_COLS;
            const uint32_t w_addr = smem_u32(sW + stage * W_BYTES);
            const uint32_t x_addr = smem_u32(sX + stage * G::X_BYTES);
            const int steps = min(BK / UMMA_K, (p.K - kb * BK + UMMA_K - 1) / UMMA_K);
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k)
                if (k < steps)
                    umma_mxf4(tmem_base, make_sdesc_kmajor_sw128(w_addr + k * (UMMA_K / 2)),
                              make_sdesc_kmajor_sw128(x_addr + k * (UMMA_K / 2)), (k & 1) ? IDESC2 : IDESC0,
                              sfw_col + 4 * (k >> 1), sfw_col + 8 + 4 * (k >> 1), kb != kb0 || k != 0 ? 1u : 0u);
            issued = true;
            umma_commit(&bars->empty[stage]);
            if (++stage == G::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok) umma_commit(&bars->acc_full);
        else if (issued) {
            umma_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, nullptr, nullptr, 0);
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------------ scale writers
        const int quarter = warp & 3;
        const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_SF))) {
                ok = false;
                break;
            }
            // lane i takes bytes [16 i, 16 i + 16) of each atom: one word per 32 rows.  A
            // gated tile has Wg's rows in words 0-1 and Wu's in 2-3, both from the half of
            // their atom that the tile's 64 rows are.
            const uint4* sw = reinterpret_cast<const uint4*>(sSFW + stage * G::SFW) + lane;
            const uint4* sx = reinterpret_cast<const uint4*>(sSFX + stage * SF_BYTES) + lane;
            uint32_t v[16];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const uint4 w = sw[a * 32], x = sx[a * 32];
                if (GATED) {
                    const uint4 u = sw[64 + a * 32];
                    const bool high = wt & 1;
                    v[4 * a] = high ? w.z : w.x; v[4 * a + 1] = high ? w.w : w.y;
                    v[4 * a + 2] = high ? u.z : u.x; v[4 * a + 3] = high ? u.w : u.y;
                } else {
                    v[4 * a] = w.x; v[4 * a + 1] = w.y; v[4 * a + 2] = w.z; v[4 * a + 3] = w.w;
                }
                // A's tile is an atom's rows, their first or last 64, or the first few
                if (NT >= 128) {
                    v[8 + 4 * a] = x.x; v[9 + 4 * a] = x.y; v[10 + 4 * a] = x.z; v[11 + 4 * a] = x.w;
                } else {
                    const bool high = m0 & 64;
                    v[8 + 4 * a] = high ? x.z : x.x; v[9 + 4 * a] = high ? x.w : x.y; v[10 + 4 * a] = 0; v[11 + 4 * a] = 0;
                }
            }
            __syncwarp();
            tmem_st_32x32b_x16(t_lane + NT + stage * SF_COLS, v);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->sf_ready[stage]);
            if (++stage == G::STAGES) { stage = 0; phase ^= 1u; }
        }
        // ------------------------------------------------------------ the partial tile
        if (ok && warp_wait(&bars->acc_full, 0, abort_flag, p.status, SITE_EPI)) {
            tc_fence_after();
            float* dst = part + quarter * 32 + lane;
#pragma unroll
            for (int c = 0; c < NT; c += 16) {
                uint32_t r[16];
                __syncwarp();
                tmem_ld_32x32b_x16(t_lane + c, r);
                tmem_ld_wait_regs(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) dst[(c + i) * BW] = __uint_as_float(r[i]);
            }
        }
    }

    tc_fence_before();
    cluster_sync();                                   // every CTA's partial tile is in its shared memory
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, G::TMEM_COLS);
        if (lane == 0 && *abort_flag) atomicAdd(&p.status->drained, 1u);
    }
    if (warp >= 2) {
        // ------------------------------------------------------------ join and store: one row of A per warp and step
        const int mine = min(NT, p.M - m0);
        const uint32_t base = smem_u32(part);
        for (int r = (int)rank + (int)ranks * (warp - 2); r < mine; r += (int)ranks * 4) {
            const size_t m = (size_t)(m0 + r);
            if constexpr (!GATED) {
                const int n0 = wt * TN + lane * 4;
                float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (uint32_t k = 0; k < ranks; ++k) {
                    const float4 v = ld_cluster_v4(mapa_shared(base + (uint32_t)(r * BW + lane * 4) * 4, k));
                    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
                }
                const float f[4] = {s.x, s.y, s.z, s.w};
                if constexpr (OUT == QG_OUT_F32) {
                    float* dst = static_cast<float*>(p.C) + m * p.N + n0;
                    if (p.vec && n0 + 4 <= p.N) *reinterpret_cast<float4*>(dst) = s;
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n0 + i < p.N) dst[i] = f[i];
                } else {
                    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.C) + m * p.N + n0;
                    if (p.vec && n0 + 4 <= p.N) {
                        const __nv_bfloat162 a = __floats2bfloat162_rn(s.x, s.y), b = __floats2bfloat162_rn(s.z, s.w);
                        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                                    *reinterpret_cast<const uint32_t*>(&b));
                    } else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n0 + i < p.N) dst[i] = __float2bfloat16_rn(f[i]);
                }
            } else {
                const int n0 = wt * TN + lane * 2;
                float2 g = make_float2(0.0f, 0.0f), u = g;
                for (uint32_t k = 0; k < ranks; ++k) {
                    const uint32_t at = mapa_shared(base + (uint32_t)(r * BW + lane * 2) * 4, k);
                    const float2 a = ld_cluster_v2(at), b = ld_cluster_v2(at + BW / 2 * 4);
                    g.x += a.x; g.y += a.y; u.x += b.x; u.y += b.y;
                }
                const float f0 = gated<ACT, OUT != QG_OUT_F32>(g.x, u.x), f1 = gated<ACT, OUT != QG_OUT_F32>(g.y, u.y);
                if constexpr (OUT == QG_OUT_MXFP4) {
                    // sixteen lanes hold one block of the result
                    uint32_t amax = max(__float_as_uint(f0) & 0x7FFFFFFFu, __float_as_uint(f1) & 0x7FFFFFFFu);
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                    const uint32_t s = scale_byte(amax);
                    const float inv = inv_scale(s == 255 ? 0 : s);
                    const uint32_t two = s == 255 ? 0u : pack2(f0 * inv, f1 * inv);
                    if (n0 < p.N) {
                        static_cast<uint8_t*>(p.C)[m * (size_t)(p.N / 2) + n0 / 2] = (uint8_t)two;
                        if ((lane & 15) == 0)
                            p.SFC[sf_offset((int)m, n0 / BLOCK, (p.N + ATOM_K - 1) / ATOM_K)] = (uint8_t)s;
                    }
                } else if constexpr (OUT == QG_OUT_F32) {
                    float* dst = static_cast<float*>(p.C) + m * p.N + n0;
                    if (n0 < p.N) dst[0] = f0;
                    if (n0 + 1 < p.N) dst[1] = f1;
                } else {
                    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.C) + m * p.N + n0;
                    if (p.vec && n0 + 2 <= p.N) *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(f0, f1);
                    else {
                        if (n0 < p.N) dst[0] = __float2bfloat16_rn(f0);
                        if (n0 + 1 < p.N) dst[1] = __float2bfloat16_rn(f1);
                    }
                }
            }
        }
        if constexpr (OUT == QG_OUT_MXFP4) {
            // zero scales where the result's atoms reach past M and N
            if (rank == 0) {
                const int blocks = p.N / BLOCK, chunks = (p.N + ATOM_K - 1) / ATOM_K;
                const bool last_x = (wt + 1) * TN >= p.N, last_y = m0 + NT >= p.M;
                const int j0 = wt * 2, nj = (last_x ? 4 * chunks : j0 + 2) - j0;
                const int rows_end = last_y ? (p.M + 127) / 128 * 128 : m0 + NT;
                for (int i = (int)threadIdx.x - 64; i < (rows_end - m0) * nj; i += 128) {
                    const int r = m0 + i / nj, j = j0 + i % nj;
                    if (r >= p.M || j >= blocks) p.SFC[sf_offset(r, j, chunks)] = 0;
                }
            }
        }
    }
    cluster_sync();                                   // nobody leaves while its partial tile is being read
}

template <int NT, int OUT, int ACT>
static int launch_nt(const void* X, const void* W, const void* W2, Params p, int split, cudaStream_t stream) {
    constexpr bool GATED = ACT >= 0;
    using G = Cfg<NT, GATED>;
    constexpr int TN = GATED ? BW / 2 : BW;
    int rc;
    if ((rc = device_status_ptr(&p.status))) return rc;
    const uint64_t row = (uint64_t)p.K / 2;
    CUtensorMap tmX, tmW, tmW2;
    if ((rc = make_tmap_2d(&tmX, X, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, (uint64_t)p.M, row, BK_BYTES, NT,
                           CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    if ((rc = make_tmap_2d(&tmW, W, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, (uint64_t)p.N, row, BK_BYTES, TN,
                           CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    tmW2 = tmW;
    if (GATED && (rc = make_tmap_2d(&tmW2, W2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, row, (uint64_t)p.N, row, BK_BYTES, TN,
                                    CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
    QG_CUDA(cudaFuncSetAttribute(rows_kernel<NT, OUT, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
    QG_CUDA(launch_overlapped(rows_kernel<NT, OUT, ACT>,
                              dim3((unsigned)(ceil_div(p.N, TN) * split), (unsigned)ceil_div(p.M, NT)), dim3(THREADS),
                              G::SMEM, stream, (unsigned)split, tmX, tmW, tmW2, p));
    return QG_OK;
}

template <int OUT, int ACT>
static int launch(const void* X, const void* W, const void* W2, const Params& p, int sms, cudaStream_t stream) {
    const int tiles_n = ceil_div(p.N, ACT >= 0 ? BW / 2 : BW);
    const int split = few_rows::pick_split(p.M, tiles_n, ceil_div(p.K, BK), sms);
    switch (few_rows::row_tile(p.M, tiles_n, sms)) {
        case 16: return launch_nt<16, OUT, ACT>(X, W, W2, p, split, stream);
        case 32: return launch_nt<32, OUT, ACT>(X, W, W2, p, split, stream);
        case 64: return launch_nt<64, OUT, ACT>(X, W, W2, p, split, stream);
        default: return launch_nt<128, OUT, ACT>(X, W, W2, p, split, stream);
    }
}

} // namespace rows

// Up to 64 rows (32 of a gated product, whose tiles are half as wide), few tiles, or
// K split four ways or more, which pays for its own start and join.  Measured, few
// rows / single / pairs: 64x28672x8192 24.6 / 25.6 / 30.3 us, 128x28672x8192 28.2 / 27.8 /
// 33.2; 256x1024x512 4.5 / 4.8 / -, 512x1024x2048 6.1 / 7.0 / -, 128x4096x4096 6.9 / 6.8
// (few tiles); 256x1024x8192 8.8 / 14.9 / 14.2, 256x4096x4096 9.1 / 9.7 / 9.9 (split in
// eight, four); 192x8192x8192 16.7 / 17.9 / 15.9, 512x4096x14336 21.4 / - / 22.4,
// 256x4096x1024 7.1 / 5.6 / 6.5 (neither); gated 64x14336x4096 16.5 / 15.5 / 19.5,
// 128x14336x4096 19.0 / 16.7 / 20.4.
bool use_rows(int M, int N, int K, bool is_gated, int sms) {
    const int tiles_n = ceil_div(N, is_gated ? rows::BW / 2 : rows::BW);
    return M <= (is_gated ? 32 : 64) || few_rows::few_tiles(M, tiles_n, sms) ||
           few_rows::pick_split(M, tiles_n, ceil_div(K, rows::BK), sms) >= 4;
}

int gemm_rows(const void* X, const void* SFX, const void* W, const void* SFW, const void* W2, const void* SFW2, void* C,
              void* SFC, int out_type, int act, bool vec, int M, int N, int K, int sms, cudaStream_t stream) {
    const rows::Params p{M, N, K, static_cast<const uint8_t*>(SFX), static_cast<const uint8_t*>(SFW),
                         static_cast<const uint8_t*>(SFW2), C, static_cast<uint8_t*>(SFC), nullptr, vec};
    if (act < 0)
        return out_type == QG_OUT_F32 ? rows::launch<QG_OUT_F32, -1>(X, W, W2, p, sms, stream)
                                      : rows::launch<QG_OUT_BF16, -1>(X, W, W2, p, sms, stream);
    if (act == QG_ACT_SILU)
        return out_type == QG_OUT_F32    ? rows::launch<QG_OUT_F32, QG_ACT_SILU>(X, W, W2, p, sms, stream)
               : out_type == QG_OUT_BF16 ? rows::launch<QG_OUT_BF16, QG_ACT_SILU>(X, W, W2, p, sms, stream)
                                         : rows::launch<QG_OUT_MXFP4, QG_ACT_SILU>(X, W, W2, p, sms, stream);
    return out_type == QG_OUT_F32    ? rows::launch<QG_OUT_F32, QG_ACT_GELU_TANH>(X, W, W2, p, sms, stream)
           : out_type == QG_OUT_BF16 ? rows::launch<QG_OUT_BF16, QG_ACT_GELU_TANH>(X, W, W2, p, sms, stream)
                                     : rows::launch<QG_OUT_MXFP4, QG_ACT_GELU_TANH>(X, W, W2, p, sms, stream);
}

} // namespace mx
} // namespace qg
