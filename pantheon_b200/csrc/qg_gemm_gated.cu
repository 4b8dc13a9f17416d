// qg_gemm_gated.cu -- the gated feed-forward projections in bf16 or fp16, and
// their backward pass, on the sm_100a tensor cores (tcgen05.mma kind::f16).
//
//   forward    G = X Wg^T, U = X Wu^T, H = act(G) * U     (one kernel)
//   backward   dG = dH * U * act'(G), dU = dH * act(G)    (a stream over M x N)
//              dX = dG Wg + dU Wu                          (contraction over 2 N)
//              dWg = dG^T X, dWu = dU^T X                  (contraction over M)
//
// All three products are one kernel over CTA pairs (clusters of two, 256 x 256
// accumulators, tcgen05.mma.cta_group::2 M=256 N=256 K=16 issued by the even
// CTA; each CTA loads its 128 rows of A and its 128 rows of B per 64-deep
// block, 32 KB, into a 6-stage ring; two accumulators in TMEM, so a tile's
// epilogue runs under the next tile's products).  The modes differ in what the
// operands are:
//   FWD   A = X; of B's 256 rows the even CTA holds 128 rows of Wg and the odd
//         CTA the same rows of Wu, so gate and up of an output lie in one TMEM
//         lane, 128 columns apart, and the epilogue joins them in registers.
//   DX    A = dG then dU along the contraction; B = Wg then Wu, whose
//         contraction index is the row: B is read column-major ("MN-major").
//   DW    A = dG or dU and B = X, both read MN-major: the contraction runs over
//         the rows of all of them, so nothing is transposed in memory.
// dG and dU are rounded to the operands' type (the tensor cores take no more):
// an error of half a step in each, of the size of the output's own rounding.
// G and U as kept are rounded likewise; H comes from the unrounded sums.
// All barrier waits are bounded (qg_ptx.cuh).
#include "qg_common.cuh"
#include "qg_formats.cuh"
#include "qg_gated.cuh"
#include "qg_launch.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace qg {
namespace ffn {

enum : int { FWD = 0, DX = 1, DW = 2 };

constexpr int BM = 128;                     // rows of A per CTA
constexpr int BN = 256;                     // accumulator columns (rows of B per pair)
constexpr int BK = 64;                      // contraction elements per stage: 128 bytes
constexpr int UMMA_K = 16;
constexpr int STAGES = 6;
constexpr int OP_BYTES = 128 * BK * 2;      // 16 KB: either operand of a CTA
constexpr int STAGE_BYTES = 2 * OP_BYTES;
constexpr int MN_BLOCK = 64 * BK * 2;       // 8 KB: 64 columns x 64 contraction rows of an MN-major operand
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
constexpr int THREADS = 256;
constexpr int EPI_WARP0 = 4;
constexpr int GROUP_M = 8;                  // row-tiles that share B's tiles in L2 (the bf16 product's best)

constexpr uint32_t SITE_PRODUCER = 0x00070001u;
constexpr uint32_t SITE_MMA_FULL = 0x00070002u;
constexpr uint32_t SITE_MMA_TMEM = 0x00070003u;
constexpr uint32_t SITE_EPI = 0x00070004u;

struct Barriers {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

struct Params {
    int rows, cols;         // of each output: FWD M x N, DX M x K, DW N x K
    int k_blocks;           // 64-deep blocks per operand pair (DX: of dG Wg; as many again of dU Wu)
    int tiles_m, tiles_n;   // DW: the row-tiles of dWg, then those of dWu
    void* out0;             // H, dX or dWg
    void* out1;             // G (or null) or dWu
    void* out2;             // U (or null)
    DeviceStatus* status;
};

__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int& mt, int& nt) {
    const int group = GROUP_M * tiles_n;
    const int g = t / group;
    const int first_m = g * GROUP_M;
    const int gm = min(tiles_m - first_m, GROUP_M);
    const int r = t - g * group;
    mt = first_m + r % gm;
    nt = r / gm;
}

// Descriptor of an MN-major operand tile: blocks of 64 elements (128 bytes)
// along MN x BK contraction rows of 128 bytes each, 128-byte swizzled as TMA
// stores them.  LBO = bytes from one 64-element block to the next, SBO = bytes
// between groups of eight contraction rows.
__device__ __forceinline__ uint64_t make_sdesc_mnmajor_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
    d |= (uint64_t)((uint32_t)MN_BLOCK >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

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

// 32 values of row `row` from column n0 on; `cols` is a multiple of 8 and rows start on 16 bytes.
template <typename T>
__device__ __forceinline__ void store32(void* out, size_t row, int n0, int cols, const float (&f)[32]) {
    T* dst = static_cast<T*>(out) + row * cols + n0;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        if (n0 + i < cols)
            *reinterpret_cast<uint4*>(dst + i) =
                make_uint4(Pack<T>::two(f[i], f[i + 1]), Pack<T>::two(f[i + 2], f[i + 3]),
                           Pack<T>::two(f[i + 4], f[i + 5]), Pack<T>::two(f[i + 6], f[i + 7]));
}

template <typename T, int MODE, int ACT>
__global__ void __launch_bounds__(THREADS, 1)
gated_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
             const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1, Params p) {
    constexpr bool A_MN = MODE == DW, B_MN = MODE != FWD;
    constexpr uint32_t FMT = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t IDESC = make_idesc(1, FMT, FMT, 2 * BM, BN) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * OP_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + STAGES * STAGE_BYTES);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int tiles = p.tiles_m * p.tiles_n;
    const int half_m = p.tiles_m / 2;                       // DW: where dWu's tiles begin
    const int nk = MODE == DX ? 2 * p.k_blocks : p.k_blocks;
    const int pair = blockIdx.x >> 1;
    const int pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(&bars->tmem_full[a], 1); mbar_init(&bars->tmem_empty[a], 8); }
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmA0);
        tma_prefetch_desc(&tmB0);
        if (MODE != FWD) tma_prefetch_desc(&tmA1);
        if (MODE != DW) tma_prefetch_desc(&tmB1);
    }
    if (warp == 2) {
        tmem_alloc_pair(&bars->tmem_base, 2 * BN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    volatile int* abort_flag = &bars->abort;
    wait_previous_grid();

    if (warp == 0 && lane == 0) {
        // ------------------------------------------------------------ producer (both CTAs)
        uint32_t stage = 0, phase = 0, armed = 0, armed_phase = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs) {
            int mt, nt;
            tile_coords(t, p.tiles_m, p.tiles_n, mt, nt);
            const bool up = MODE == DW && mt >= half_m;      // a tile of dWu
            const int m0 = (MODE == DW ? mt - (up ? half_m : 0) : mt) * 2 * BM + (int)rank * BM;
            const int n0 = MODE == FWD ? nt * 128 : nt * BN + (int)rank * 128;
            for (int kb = 0; kb < nk; ++kb) {
                if (!mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
                if (leader) mbar_arrive_expect_tx(&bars->full[stage], 2 * STAGE_BYTES);
                const uint32_t full = mapa_shared(smem_u32(&bars->full[stage]), 0);
                const bool second = MODE == DX && kb >= p.k_blocks;   // dU and Wu
                const int k0 = (second ? kb - p.k_blocks : kb) * BK;
                const CUtensorMap* a = up || second ? &tmA1 : &tmA0;
                const CUtensorMap* b = (MODE == FWD && !leader) || second ? &tmB1 : &tmB0;
                uint8_t* da = sA + stage * OP_BYTES;
                uint8_t* db = sB + stage * OP_BYTES;
                // x coordinates are in bytes (the maps describe byte matrices)
                if constexpr (A_MN) {
                    tma_load_2d_pair(da, a, full, m0 * 2, k0);
                    tma_load_2d_pair(da + MN_BLOCK, a, full, m0 * 2 + 128, k0);
                } else {
                    tma_load_2d_pair(da, a, full, k0 * 2, m0);
                }
                if constexpr (B_MN) {
                    tma_load_2d_pair(db, b, full, n0 * 2, k0);
                    tma_load_2d_pair(db + MN_BLOCK, b, full, n0 * 2 + 128, k0);
                } else {
                    tma_load_2d_pair(db, b, full, k0 * 2, n0);
                }
                armed |= 1u << stage;
                armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        if (!ok && leader) {
            // copies of both CTAs complete on these barriers: let them land
            for (int s = 0; s < STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
        }
    } else if (warp == 1 && lane == 0 && leader) {
        // ------------------------------------------------------------ MMA issuer (even CTA)
        uint32_t stage = 0, phase = 0;
        bool ok = true, issued = false;
        int iter = 0;
        for (int t = pair; t < tiles && ok; t += pairs, ++iter) {
            const uint32_t acc = iter & 1;
            const uint32_t acc_phase = (iter >> 1) & 1;
            if (!mbar_wait(&bars->tmem_empty[acc], acc_phase ^ 1u, abort_flag, p.status, SITE_MMA_TMEM)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + acc * BN;
            for (int kb = 0; kb < nk; ++kb) {
                if (!mbar_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_MMA_FULL)) { ok = false; break; }
                tc_fence_after();
                const uint32_t a_addr = smem_u32(sA + stage * OP_BYTES);
                const uint32_t b_addr = smem_u32(sB + stage * OP_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k) {
                    // 16 contraction elements: 32 bytes of a K-major row, 16 rows of an MN-major tile
                    const uint64_t ad = A_MN ? make_sdesc_mnmajor_sw128(a_addr + k * UMMA_K * 128)
                                             : make_sdesc_kmajor_sw128(a_addr + k * UMMA_K * 2);
                    const uint64_t bd = B_MN ? make_sdesc_mnmajor_sw128(b_addr + k * UMMA_K * 128)
                                             : make_sdesc_kmajor_sw128(b_addr + k * UMMA_K * 2);
                    umma_f16_pair(d_tmem, ad, bd, IDESC, (kb | k) != 0 ? 1u : 0u);
                }
                issued = true;
                const uint32_t e = smem_u32(&bars->empty[stage]);
                umma_commit_pair(mapa_shared(e, 0));
                umma_commit_pair(mapa_shared(e, 1));
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (ok) {
                const uint32_t f = smem_u32(&bars->tmem_full[acc]);
                umma_commit_pair(mapa_shared(f, 0));
                umma_commit_pair(mapa_shared(f, 1));
            }
        }
        if (!ok && issued) {
            umma_commit_pair(mapa_shared(smem_u32(&bars->drain), 0));
            mbar_wait(&bars->drain, 0, nullptr, nullptr, 0);
        }
    } else if (warp >= EPI_WARP0) {
        // ------------------------------------------------------------ epilogue (both CTAs)
        const int ew = warp - EPI_WARP0;
        int iter = 0;
        for (int t = pair; t < tiles; t += pairs, ++iter) {
            int mt, nt;
            tile_coords(t, p.tiles_m, p.tiles_n, mt, nt);
            const uint32_t acc = iter & 1;
            const uint32_t acc_phase = (iter >> 1) & 1;
            int ok = 1;
            if (lane == 0) ok = mbar_wait(&bars->tmem_full[acc], acc_phase, abort_flag, p.status, SITE_EPI) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            tc_fence_after();
            const bool up = MODE == DW && mt >= half_m;
            const int m = (MODE == DW ? mt - (up ? half_m : 0) : mt) * 2 * BM + (int)rank * BM + ew * 32 + lane;
            const bool row_ok = m < p.rows;
            const uint32_t t_row = tmem_base + ((uint32_t)(ew * 32) << 16) + acc * BN;
            if constexpr (MODE == FWD) {
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    uint32_t rg[32], ru[32];
                    __syncwarp();
                    tmem_ld_32x32b_x32(t_row + c, rg);
                    tmem_ld_32x32b_x32(t_row + 128 + c, ru);
                    tmem_ld_wait_regs(rg);
                    tmem_ld_wait_regs(ru);
                    const int n0 = nt * 128 + c;
                    if (!row_ok || n0 >= p.cols) continue;
                    float f[32];
                    if (p.out1) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(rg[i]);
                        store32<T>(p.out1, m, n0, p.cols, f);
#pragma unroll
                        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(ru[i]);
                        store32<T>(p.out2, m, n0, p.cols, f);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) f[i] = gated<ACT, true>(__uint_as_float(rg[i]), __uint_as_float(ru[i]));
                    store32<T>(p.out0, m, n0, p.cols, f);
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < BN; c += 32) {
                    uint32_t r[32];
                    __syncwarp();
                    tmem_ld_32x32b_x32(t_row + c, r);
                    tmem_ld_wait_regs(r);
                    const int n0 = nt * BN + c;
                    if (!row_ok || n0 >= p.cols) continue;
                    float f[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
                    store32<T>(up ? p.out1 : p.out0, m, n0, p.cols, f);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&bars->tmem_empty[acc]), 0));
        }
    }

    // the even CTA's MMAs read this CTA's shared memory and write its TMEM:
    // neither CTA frees anything before both are done
    tc_fence_before();
    cluster_sync();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 2 * BN);
        if (lane == 0 && *abort_flag) atomicAdd(&p.status->drained, 1u);
    }
}

// dG = dH * U * act'(G), dU = dH * act(G), eight elements per thread and step.
// Five streams of 2 bytes per element: bound by memory.
template <typename T, int ACT>
__global__ void __launch_bounds__(256)
gate_backward_kernel(const uint4* __restrict__ dH, const uint4* __restrict__ G, const uint4* __restrict__ U,
                     uint4* __restrict__ dG, uint4* __restrict__ dU, uint64_t n8) {
    const uint64_t step = (uint64_t)gridDim.x * blockDim.x;
    wait_previous_grid();
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += step) {
        const uint4 vh = __ldg(dH + i), vg = __ldg(G + i), vu = __ldg(U + i);
        const uint32_t h[4] = {vh.x, vh.y, vh.z, vh.w}, g[4] = {vg.x, vg.y, vg.z, vg.w}, u[4] = {vu.x, vu.y, vu.z, vu.w};
        uint32_t og[4], ou[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 fh = Pack<T>::unpack(h[j]), fg = Pack<T>::unpack(g[j]), fu = Pack<T>::unpack(u[j]);
            float a0, s0, a1, s1;
            gate_slope<ACT>(fg.x, a0, s0);
            gate_slope<ACT>(fg.y, a1, s1);
            og[j] = Pack<T>::two(fh.x * fu.x * s0, fh.y * fu.y * s1);
            ou[j] = Pack<T>::two(fh.x * a0, fh.y * a1);
        }
        dG[i] = make_uint4(og[0], og[1], og[2], og[3]);
        dU[i] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
    }
}

// The byte matrix of a 2-byte tensor [rows, cols] in boxes of 128 bytes x box_rows.
static int make_map(CUtensorMap* map, const void* base, int rows, int cols, int box_rows) {
    return make_tmap_2d(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)cols * 2, (uint64_t)rows,
                        (uint64_t)cols * 2, 128, (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int MODE, int ACT>
static int launch(const CUtensorMap& a0, const CUtensorMap& a1, const CUtensorMap& b0, const CUtensorMap& b1, Params p,
                  cudaStream_t stream) {
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
    if ((rc = device_status_ptr(&p.status))) return rc;
    QG_CUDA(cudaFuncSetAttribute(gated_kernel<T, MODE, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    // persistent pairs: as many as can be resident at once
    static int resident[64] = {};
    int dev = 0;
    QG_CUDA(cudaGetDevice(&dev));
    int res = resident[dev & 63];
    if (!res) {
        cudaLaunchConfig_t lc = {};
        lc.gridDim = dim3(info->sm_count & ~1);
        lc.blockDim = dim3(THREADS);
        lc.dynamicSmemBytes = SMEM_BYTES;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {2, 1, 1};
        lc.attrs = at;
        lc.numAttrs = 1;
        QG_CUDA(cudaOccupancyMaxActiveClusters(&res, gated_kernel<T, MODE, ACT>, &lc));
        if (res < 1) res = 1;
        resident[dev & 63] = res;
    }
    const int tiles = p.tiles_m * p.tiles_n;
    const int pairs = tiles < res ? tiles : res;
    QG_CUDA(launch_overlapped(gated_kernel<T, MODE, ACT>, dim3(2 * pairs), dim3(THREADS), SMEM_BYTES, stream, 2, a0, a1, b0,
                              b1, p));
    return QG_OK;
}

static int check_shape(const char* name, int M, int N, int K) {
    QG_CHECK_ARG(M > 0 && N > 0 && K > 0, "%s: empty shape %dx%dx%d", name, M, N, K);
    QG_CHECK_ARG(N % 8 == 0 && K % 8 == 0, "%s: N=%d and K=%d must be multiples of 8 (16-byte rows)", name, N, K);
    // x coordinates are bytes in 32 bits; tile counts fit too
    QG_CHECK_ARG(M <= (1 << 29) && N <= (1 << 29) && K <= (1 << 29), "%s: shape %dx%dx%d is too large", name, M, N, K);
    const int64_t m = ceil_div(M, 256), n = ceil_div(N, 128), k = ceil_div(K, 256);
    QG_CHECK_ARG(m * n <= (1 << 30) && m * k <= (1 << 30) && n * k <= (1 << 30), "%s: shape %dx%dx%d is too large", name, M, N, K);
    return QG_OK;
}

template <typename T>
static int forward(const char* name, const void* X, const void* Wg, const void* Wu, void* H, void* G, void* U, int act,
                   int M, int N, int K, cudaStream_t stream) {
    QG_CHECK_ARG(X && Wg && Wu && H, "%s: null operand or output", name);
    QG_CHECK_ARG((G == nullptr) == (U == nullptr), "%s: G and U are kept together or not at all", name);
    QG_CHECK_ARG(act == QG_ACT_SILU || act == QG_ACT_GELU_TANH, "%s: unknown activation %d", name, act);
    int rc = check_shape(name, M, N, K);
    if (rc) return rc;
    QG_CHECK_ARG((((uintptr_t)X | (uintptr_t)Wg | (uintptr_t)Wu | (uintptr_t)H | (uintptr_t)G | (uintptr_t)U) & 15) == 0,
                 "%s: operands and outputs must be 16-byte aligned", name);
    CUtensorMap a, b0, b1;
    if ((rc = make_map(&a, X, M, K, BM)) || (rc = make_map(&b0, Wg, N, K, 128)) || (rc = make_map(&b1, Wu, N, K, 128)))
        return rc;
    Params p{M, N, ceil_div(K, BK), ceil_div(M, 2 * BM), ceil_div(N, 128), H, G, U, nullptr};
    return act == QG_ACT_SILU ? launch<T, FWD, QG_ACT_SILU>(a, a, b0, b1, p, stream)
                              : launch<T, FWD, QG_ACT_GELU_TANH>(a, a, b0, b1, p, stream);
}

template <typename T>
static int backward(const char* name, const void* dH, const void* X, const void* Wg, const void* Wu, const void* G,
                    const void* U, void* dX, void* dWg, void* dWu, int act, int M, int N, int K, void* workspace,
                    uint64_t workspace_bytes, cudaStream_t stream) {
    QG_CHECK_ARG(dH && X && Wg && Wu && G && U, "%s: null operand", name);
    QG_CHECK_ARG((dWg == nullptr) == (dWu == nullptr), "%s: dWg and dWu are computed together or not at all", name);
    QG_CHECK_ARG(dX || dWg, "%s: no gradient asked for", name);
    QG_CHECK_ARG(act == QG_ACT_SILU || act == QG_ACT_GELU_TANH, "%s: unknown activation %d", name, act);
    int rc = check_shape(name, M, N, K);
    if (rc) return rc;
    const uint64_t one = (uint64_t)M * (uint64_t)N * 2;           // a multiple of 16
    QG_CHECK_ARG(workspace && workspace_bytes >= 2 * one, "%s: workspace of %llu bytes, %llu needed", name,
                 (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)(2 * one));
    QG_CHECK_ARG((((uintptr_t)dH | (uintptr_t)X | (uintptr_t)Wg | (uintptr_t)Wu | (uintptr_t)G | (uintptr_t)U |
                   (uintptr_t)dX | (uintptr_t)dWg | (uintptr_t)dWu | (uintptr_t)workspace) & 15) == 0,
                 "%s: operands, outputs and workspace must be 16-byte aligned", name);
    DeviceInfo* info = nullptr;
    if ((rc = current_device_info(&info))) return rc;
    void* dG = workspace;
    void* dU = static_cast<uint8_t*>(workspace) + one;
    const uint64_t n8 = one / 16, blocks = (n8 + 255) / 256, most = (uint64_t)info->sm_count * 8;
    const int grid = (int)(blocks < most ? blocks : most);
    auto* vh = static_cast<const uint4*>(dH);
    auto* vg = static_cast<const uint4*>(G);
    auto* vu = static_cast<const uint4*>(U);
    auto* og = static_cast<uint4*>(dG);
    auto* ou = static_cast<uint4*>(dU);
    QG_CUDA(launch_overlapped(act == QG_ACT_SILU ? gate_backward_kernel<T, QG_ACT_SILU>
                                                 : gate_backward_kernel<T, QG_ACT_GELU_TANH>,
                              dim3(grid), dim3(256), 0, stream, 1, vh, vg, vu, og, ou, n8));
    CUtensorMap a0, a1, b0, b1;
    if (dX) {
        if ((rc = make_map(&a0, dG, M, N, BM)) || (rc = make_map(&a1, dU, M, N, BM)) ||
            (rc = make_map(&b0, Wg, N, K, BK)) || (rc = make_map(&b1, Wu, N, K, BK)))
            return rc;
        Params p{M, K, ceil_div(N, BK), ceil_div(M, 2 * BM), ceil_div(K, BN), dX, nullptr, nullptr, nullptr};
        if ((rc = launch<T, DX, QG_ACT_SILU>(a0, a1, b0, b1, p, stream))) return rc;
    }
    if (dWg) {
        if ((rc = make_map(&a0, dG, M, N, BK)) || (rc = make_map(&a1, dU, M, N, BK)) || (rc = make_map(&b0, X, M, K, BK)))
            return rc;
        Params p{N, K, ceil_div(M, BK), 2 * ceil_div(N, 2 * BM), ceil_div(K, BN), dWg, dWu, nullptr, nullptr};
        if ((rc = launch<T, DW, QG_ACT_SILU>(a0, a1, b0, b0, p, stream))) return rc;
    }
    return QG_OK;
}

} // namespace ffn
} // namespace qg

extern "C" int qg_gemm_gated_bf16(const void* X, const void* Wg, const void* Wu, void* H, void* G, void* U, int act,
                                  int M, int N, int K, void* stream) {
    return qg::ffn::forward<__nv_bfloat16>("qg_gemm_gated_bf16", X, Wg, Wu, H, G, U, act, M, N, K,
                                           static_cast<cudaStream_t>(stream));
}

extern "C" int qg_gemm_gated_f16(const void* X, const void* Wg, const void* Wu, void* H, void* G, void* U, int act,
                                 int M, int N, int K, void* stream) {
    return qg::ffn::forward<__half>("qg_gemm_gated_f16", X, Wg, Wu, H, G, U, act, M, N, K,
                                    static_cast<cudaStream_t>(stream));
}

extern "C" int qg_gemm_gated_backward_workspace_bytes(int M, int N, uint64_t* bytes) {
    QG_CHECK_ARG(bytes && M > 0 && N > 0, "qg_gemm_gated_backward_workspace_bytes: bad argument");
    *bytes = 4ull * (uint64_t)M * (uint64_t)N;
    return QG_OK;
}

extern "C" int qg_gemm_gated_bf16_backward(const void* dH, const void* X, const void* Wg, const void* Wu, const void* G,
                                           const void* U, void* dX, void* dWg, void* dWu, int act, int M, int N, int K,
                                           void* workspace, uint64_t workspace_bytes, void* stream) {
    return qg::ffn::backward<__nv_bfloat16>("qg_gemm_gated_bf16_backward", dH, X, Wg, Wu, G, U, dX, dWg, dWu, act, M, N,
                                            K, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int qg_gemm_gated_f16_backward(const void* dH, const void* X, const void* Wg, const void* Wu, const void* G,
                                          const void* U, void* dX, void* dWg, void* dWu, int act, int M, int N, int K,
                                          void* workspace, uint64_t workspace_bytes, void* stream) {
    return qg::ffn::backward<__half>("qg_gemm_gated_f16_backward", dH, X, Wg, Wu, G, U, dX, dWg, dWu, act, M, N, K,
                                     workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
