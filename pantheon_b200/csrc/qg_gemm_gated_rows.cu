// qg_gemm_gated_rows.cu -- the forward pass and dX of qg_gemm_gated.cu for few rows
// of X (decode steps, short prompts; more rows where a long contraction meets few
// tiles), where reading the weights once is the whole cost: 4 N K bytes.
//
// As in qg_gemm_mxfp4_rows.cu the operands change places: the weights are the M
// side of tcgen05.mma, 128 to a tile, and NT = 16, 32, 64 or 128 rows of X (dG, dU)
// its N side.  The contraction is split over the CTAs of a cluster (1 to 8); each
// sums its part in TMEM, puts the partial tile in its shared memory, and every
// CTA of the cluster joins a share of the rows from all of them over
// distributed shared memory, in rank order: no workspace, no atomics, the same
// bits on every run.
//   forward   a tile's weights are 64 rows of Wg and the same 64 of Wu
//   dX        128 columns of Wg, then of Wu along the contraction (2 N): the weights
//             are read MN-major.  dG and dU in two terms (PARTS) bring their
//             remainders beside them in a stage.
//
// Bound by the weights' bytes: measured (bf16) 1x8192x4096 22.7 us (134 MB, 5.9 TB/s,
// 0.90 of the measured copy bandwidth), 16x8192x4096 23.7, 64x8192x4096 25.7,
// 1x4096x4096 13.4, 1x1024x1024 3.8; dX 1x8192x4096 26.0 with its stream over M x N,
// 64x8192x4096 28.4.  What is left is a launch's start and end, 2-3 us.
//
// 192 threads, two CTAs per SM:
//   warp 0      producer: TMA loads per 64-element K block, into a ring of up to 105 KB.
//   warp 1      TMEM allocator and MMA issuer (M=128 N=NT K=16).
//   warps 2-5   epilogue.
// All barrier waits are bounded (qg_ptx.cuh).
#include "qg_common.cuh"
#include "qg_few_rows.cuh"
#include "qg_formats.cuh"
#include "qg_gated.cuh"
#include "qg_launch.cuh"
#include "qg_mxfp4_mma.cuh"
#include "qg_rows.cuh"

#include <type_traits>

namespace qg {
namespace ffn {
namespace rows {

using mx::warp_wait;

constexpr int BW = 128;                        // weight rows (dX: columns) of a tile
constexpr int BK = 64;
constexpr int BK_BYTES = BK * 2;
constexpr int UMMA_K = 16;
constexpr int W_BYTES = BW * BK_BYTES;         // 16 KB
constexpr int THREADS = 192;

constexpr int DX = -1;                         // in place of the activation

template <int NT, int PARTS>
struct Cfg {
    static constexpr int X_BYTES = NT * BK_BYTES;           // of one term
    static constexpr int STAGE = W_BYTES + PARTS * X_BYTES;
    static constexpr int STAGES = 105 * 1024 / STAGE;       // two CTAs share an SM's 227 KB
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
    static constexpr int TMEM_COLS = NT < 32 ? 32 : NT;
    static_assert(NT * BW * 4 <= STAGES * STAGE, "the partial tile fits the ring");
};

constexpr uint32_t SITE_PRODUCER = 0x00090001u;
constexpr uint32_t SITE_MMA_FULL = 0x00090002u;
constexpr uint32_t SITE_EPI = 0x00090003u;

struct Maps {
    CUtensorMap w[2];         // Wg, Wu
    CUtensorMap x[2][2];      // X; dX: [dG, dU][value, remainder]
};

struct Params {
    int M, N, K;
    void* out;                // H, or dX
    void* G;                  // or null
    void* U;
    DeviceStatus* status;
};

template <int MAX>
struct Barriers {
    uint64_t full[MAX];
    uint64_t empty[MAX];
    uint64_t acc_full;
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

template <typename T, int NT, int ACT, int PARTS>
__global__ void __launch_bounds__(THREADS, 2)
gated_rows_kernel(const __grid_constant__ Maps maps, Params p) {
    constexpr bool BACK = ACT == DX;
    using C = Cfg<NT, PARTS>;
    constexpr int TN = BACK ? BW : BW / 2;           // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t* sW = smem;
    uint8_t* sX = sW + C::STAGES * W_BYTES;
    using Bars = Barriers<C::STAGES>;
    static_assert(sizeof(Bars) <= 256, "barrier block");
    Bars* bars = reinterpret_cast<Bars*>(smem + C::STAGES * C::STAGE);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();
    const int n_tile = (int)(blockIdx.x / ranks) * TN;
    const int m0 = blockIdx.y * NT;
    const int half = ((BACK ? p.N : p.K) + BK - 1) / BK;     // dX: blocks of dG, as many of dU
    const int nk_all = BACK ? 2 * half : half;
    const int kb0 = (int)((int64_t)nk_all * rank / ranks), kb1 = (int)((int64_t)nk_all * (rank + 1) / ranks);

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        mbar_init(&bars->acc_full, 1);
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&bars->tmem_base, C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    volatile int* abort_flag = &bars->abort;
    wait_previous_grid();
    float* part = reinterpret_cast<float*>(smem);    // [row][tile's weights], over the ring once it is drained

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ producer
        uint32_t stage = 0, phase = 0, armed = 0, armed_phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
            uint64_t* full = &bars->full[stage];
            mbar_arrive_expect_tx(full, C::STAGE);
            uint8_t* w = sW + stage * W_BYTES;
            uint8_t* x = sX + stage * PARTS * C::X_BYTES;
            if constexpr (BACK) {
                const int which = kb >= half, b = kb - which * half;
                tma_load_2d(w, &maps.w[which], full, n_tile * 2, b * BK);
                tma_load_2d(w + W_BYTES / 2, &maps.w[which], full, n_tile * 2 + 128, b * BK);
                for (int q = 0; q < PARTS; ++q)
                    tma_load_2d(x + q * C::X_BYTES, &maps.x[which][q], full, b * BK_BYTES, m0);
            } else {
                tma_load_2d(w, &maps.w[0], full, kb * BK_BYTES, n_tile);
                tma_load_2d(w + W_BYTES / 2, &maps.w[1], full, kb * BK_BYTES, n_tile);
                tma_load_2d(x, &maps.x[0][0], full, kb * BK_BYTES, m0);
            }
            armed |= 1u << stage;
            armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
        // the last releases land before the CTA's shared memory goes away
        for (int i = 0; i < C::STAGES && ok; ++i) {
            ok = mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER);
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok)
            for (int s = 0; s < C::STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
    } else if (warp == 1 && lane == 0) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t IDESC = make_idesc(1, FMT, FMT, BW, NT) | (BACK ? 1u << 15 : 0u);
        uint32_t stage = 0, phase = 0;
        bool ok = true, issued = false;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_MMA_FULL)) { ok = false; break; }
            tc_fence_after();
            const uint32_t w_addr = smem_u32(sW + stage * W_BYTES);
            const uint32_t x_addr = smem_u32(sX + stage * PARTS * C::X_BYTES);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k) {
                    const uint64_t w_desc = BACK ? make_sdesc_mnmajor_sw128(w_addr + k * (UMMA_K * 128), W_BYTES / 2)
                                                 : make_sdesc_kmajor_sw128(w_addr + k * (UMMA_K * 2));
                    umma_f16(tmem_base, w_desc, make_sdesc_kmajor_sw128(x_addr + q * C::X_BYTES + k * (UMMA_K * 2)), IDESC,
                             kb != kb0 || q != 0 || k != 0 ? 1u : 0u);
                }
            issued = true;
            umma_commit(&bars->empty[stage]);
            if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
        }
        if (ok) umma_commit(&bars->acc_full);
        else if (issued) {
            umma_commit(&bars->drain);
            mbar_wait(&bars->drain, 0, nullptr, nullptr, 0);
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------------ the partial tile
        const int quarter = warp & 3;
        if (warp_wait(&bars->acc_full, 0, abort_flag, p.status, SITE_EPI)) {
            tc_fence_after();
            const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
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
        tmem_dealloc(tmem_base, C::TMEM_COLS);
        if (lane == 0 && *abort_flag) atomicAdd(&p.status->drained, 1u);
    }
    if (warp >= 2) {
        // ------------------------------------------------------------ join and store: one row of X per warp and step
        const int mine = min(NT, p.M - m0);
        const uint32_t base = smem_u32(part);
        const int cols = BACK ? p.K : p.N;            // a multiple of 8
        const int n = n_tile + lane * (BACK ? 4 : 2);
        for (int r = (int)rank + (int)ranks * (warp - 2); r < mine; r += (int)ranks * 4) {
            const size_t at = (size_t)(m0 + r) * cols + n;
            if constexpr (BACK) {
                float4 d = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (uint32_t k = 0; k < ranks; ++k) {
                    const float4 v = ld_cluster_v4(mapa_shared(base + (uint32_t)(r * BW + lane * 4) * 4, k));
                    d.x += v.x; d.y += v.y; d.z += v.z; d.w += v.w;
                }
                if (n < cols)
                    static_cast<uint2*>(p.out)[at / 4] = make_uint2(Pack<T>::two(d.x, d.y), Pack<T>::two(d.z, d.w));
            } else {
                float2 g = make_float2(0.0f, 0.0f), u = g;
                for (uint32_t k = 0; k < ranks; ++k) {
                    const uint32_t from = mapa_shared(base + (uint32_t)(r * BW + lane * 2) * 4, k);
                    const float2 a = ld_cluster_v2(from), b = ld_cluster_v2(from + TN * 4);
                    g.x += a.x; g.y += a.y; u.x += b.x; u.y += b.y;
                }
                if (n >= cols) continue;
                if (p.G) {
                    static_cast<uint32_t*>(p.G)[at / 2] = Pack<T>::two(g.x, g.y);
                    static_cast<uint32_t*>(p.U)[at / 2] = Pack<T>::two(u.x, u.y);
                }
                static_cast<uint32_t*>(p.out)[at / 2] = Pack<T>::two(gated<ACT, true>(g.x, u.x), gated<ACT, true>(g.y, u.y));
            }
        }
    }
    cluster_sync();                                   // nobody leaves while its partial tile is being read
}

static int make_map(CUtensorMap* map, const void* base, int rows, int cols, int box_rows) {
    return make_tmap_2d(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)cols * 2, (uint64_t)rows,
                        (uint64_t)cols * 2, BK_BYTES, (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// x: X, or for dX dG and dU, then their remainders.
template <typename T, int NT, int ACT, int PARTS>
static int launch_nt(const void* const (&x)[4], const void* Wg, const void* Wu, Params p, int split, cudaStream_t stream) {
    constexpr bool BACK = ACT == DX;
    using C = Cfg<NT, PARTS>;
    int rc;
    if ((rc = device_status_ptr(&p.status))) return rc;
    Maps maps;
    if ((rc = make_map(&maps.w[0], Wg, p.N, p.K, 64)) || (rc = make_map(&maps.w[1], Wu, p.N, p.K, 64))) return rc;
    for (int i = 0; i < 4; ++i) {
        if (!x[i]) maps.x[i & 1][i >> 1] = maps.x[0][0];      // not read
        else if ((rc = make_map(&maps.x[i & 1][i >> 1], x[i], p.M, BACK ? p.N : p.K, NT))) return rc;
    }
    const auto kernel = gated_rows_kernel<T, NT, ACT, PARTS>;
    QG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    const int tiles = BACK ? ceil_div(p.K, BW) : ceil_div(p.N, BW / 2);
    QG_CUDA(launch_overlapped(kernel, dim3((unsigned)(tiles * split), (unsigned)ceil_div(p.M, NT)), dim3(THREADS),
                              C::SMEM, stream, (unsigned)split, maps, p));
    return QG_OK;
}

template <typename T, int ACT, int PARTS>
static int launch(const void* const (&x)[4], const void* Wg, const void* Wu, const Params& p, int sms,
                  cudaStream_t stream) {
    const int tiles_n = ACT == DX ? ceil_div(p.K, BW) : ceil_div(p.N, BW / 2);
    const int split = few_rows::pick_split(p.M, tiles_n, ACT == DX ? 2 * ceil_div(p.N, BK) : ceil_div(p.K, BK), sms);
    switch (few_rows::row_tile(p.M, tiles_n, sms)) {
        case 16: return launch_nt<T, 16, ACT, PARTS>(x, Wg, Wu, p, split, stream);
        case 32: return launch_nt<T, 32, ACT, PARTS>(x, Wg, Wu, p, split, stream);
        case 64: return launch_nt<T, 64, ACT, PARTS>(x, Wg, Wu, p, split, stream);
        default: return launch_nt<T, 128, ACT, PARTS>(x, Wg, Wu, p, split, stream);
    }
}

} // namespace rows

// Forward: up to 64 rows, few tiles, or K split four ways or more.  Measured (pairs / few
// rows, us): 1x1024x1024 8.7 / 3.8, 64x1024x4096 14.1 / 7.9, 64x8192x4096 28.9 / 25.7,
// 128x8192x4096 (unsplit) 29.9 / 30.5, 128x4096x4096 (four) 20.3 / 17.9, 256x4096x4096 (two)
// 20.3 / 23.3, 256x1024x512 7.0 / 6.0, 256x1024x4096 17.8 / 11.0, 512x1024x4096 18.1 / 14.4,
// 1024x1024x4096 (two) 19.5 / 21.6.
bool use_rows(int M, int N, int K, int sms) {
    const int tiles_n = ceil_div(N, rows::BW / 2);
    return M <= 64 || few_rows::few_tiles(M, tiles_n, sms) ||
           few_rows::pick_split(M, tiles_n, ceil_div(K, rows::BK), sms) >= 4;
}

int rows_split_dx(int M, int N, int K, int sms) {
    return few_rows::pick_split(M, ceil_div(K, rows::BW), 2 * ceil_div(N, rows::BK), sms);
}

int gated_rows(const void* X, const void* Wg, const void* Wu, void* H, void* G, void* U, bool half, int act, int M,
               int N, int K, int sms, cudaStream_t stream) {
    const rows::Params p{M, N, K, H, G, U, nullptr};
    const void* const x[4] = {X, nullptr, nullptr, nullptr};
    const bool silu = act == QG_ACT_SILU;
    if (half)
        return silu ? rows::launch<__half, QG_ACT_SILU, 1>(x, Wg, Wu, p, sms, stream)
                    : rows::launch<__half, QG_ACT_GELU_TANH, 1>(x, Wg, Wu, p, sms, stream);
    return silu ? rows::launch<__nv_bfloat16, QG_ACT_SILU, 1>(x, Wg, Wu, p, sms, stream)
                : rows::launch<__nv_bfloat16, QG_ACT_GELU_TANH, 1>(x, Wg, Wu, p, sms, stream);
}

int gated_rows_dx(const void* const (&d)[4], const void* Wg, const void* Wu, void* dX, bool half, int M, int N, int K,
                  int sms, cudaStream_t stream) {
    const rows::Params p{M, N, K, dX, nullptr, nullptr, nullptr};
    if (d[2])
        return half ? rows::launch<__half, rows::DX, 2>(d, Wg, Wu, p, sms, stream)
                    : rows::launch<__nv_bfloat16, rows::DX, 2>(d, Wg, Wu, p, sms, stream);
    return half ? rows::launch<__half, rows::DX, 1>(d, Wg, Wu, p, sms, stream)
                : rows::launch<__nv_bfloat16, rows::DX, 1>(d, Wg, Wu, p, sms, stream);
}

} // namespace ffn
} // namespace qg
