// qg_gemm_gated.cu -- the gated feed-forward projections in bf16 or fp16, and
// their backward pass, on the sm_100a tensor cores (tcgen05.mma kind::f16).
//
//   forward    G = X Wg^T, U = X Wu^T, H = act(G) * U     (one kernel)
//   backward   dG = dH * U * act'(G), dU = dH * act(G)    (a stream over M x N)
//              dX = dG Wg + dU Wu                          (contraction over 2 N)
//              dWg = dG^T X, dWu = dU^T X                  (contraction over M)
//                                                          (one kernel for the three,
//                                                           or dX apart with few rows)
//
// Each product is tiles of CTA pairs (256 x 256 accumulators, tcgen05.mma
// .cta_group::2 M=256 N=256 K=16 issued by the even CTA); per 64-deep contraction
// block a CTA loads its 128 rows of A and 128 of B's 256 rows (32 KB) into a
// 6-stage ring.  TMEM holds two accumulators, tile n of a pair in region n % 2;
// epilogue group n % 2 drains it under the next tile's products.  (256 x 512
// tiles, a quarter fewer bytes per product but one accumulator, measured slower:
// 403 us against 372 forward and 762 against 749 backward at 4096x8192x4096.)
// What the operands are:
//   forward   A = X; of B's 256 rows the even CTA holds 128 rows of Wg
//             and the odd CTA the same rows of Wu, so gate and up of an output lie
//             in one TMEM lane, 128 columns apart, and the epilogue joins them.
//   dX        A = dG then dU along the contraction; B = Wg then Wu, whose
//             contraction index is the row: B is read column-major ("MN-major").
//   dWg, dWu  A = dG or dU and B = X, both read MN-major: the contraction runs over
//             the rows of all of them, so nothing is transposed in memory.
// SPLIT: few tiles share the GPU better when a cluster of S pairs takes one tile
// and each pair a part of its contraction; the partial tiles meet in shared memory
// and every CTA joins a share of the columns over distributed shared memory, in
// rank order (the same bits on every run, no workspace).
// dG and dU are operands of the tensor cores, so rounded to the type: an error of
// half a step in each, of the size of the result's own rounding (gradients of
// 4096x8192x4096 are off by 0.0023 of their norm in bf16, against 0.0017 from their own
// rounding alone; fp16 0.00029 and 0.00021).  In two terms (value and remainder; a
// stage then holds both beside one block of B) that rounding is gone, at twice the
// products and the workspace.  The line between the two is a plain one of cost, M N
// <= 65536, whatever the sums' lengths (M for dWg and dWu, 2 N for dX); accuracy and
// workspace step there.  All gradients, two terms / one on the line's other side:
// 16x4096x4096 37.0 / 37.1 us (4104), 8x8192x4096 63.0 / 60.9 (8200), 256x256x1024
// 10.6 / 8.9 (264), 128x512x1024 15.0 / 11.1 (520), 1024x64x1024 14.7 / 10.3 (72),
// 1x65536x1024 154 / 134 (65544); the largest, where the products are the time, would
// take twice as long.  fp16 keeps its range in either form: what is below 2^-25 is 0.
// G and U as kept are rounded likewise; H comes from the unrounded sums.
// Few rows have a kernel of their own for forward and dX (use_rows, use_rows_dx,
// qg_gemm_gated_rows.cu).
// Bound by the tensor cores: measured at 4096x8192x4096 bf16 the forward pass takes
// 342-357 us (1.54-1.61 PFLOP/s, 0.90-0.94 of the measured rate, tensor pipe 97 %
// active), the backward pass 737-760 us (47 of them the stream over M x N, the rest at
// 98 % of the tensor pipe); back to back under the power cap 403 and 899 us.
// All barrier waits are bounded (qg_ptx.cuh).
#include "qg_common.cuh"
#include "qg_formats.cuh"
#include "qg_gated.cuh"
#include "qg_launch.cuh"
#include "qg_mxfp4_mma.cuh"
#include "qg_rows.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <atomic>
#include <type_traits>

namespace qg {
namespace ffn {

using mx::elect_one;
using mx::mbar_arrive_relaxed;
using mx::umma_commit_both;
using mx::warp_wait;

enum : int { FWD = 0, DX = 1, DW = 2 };

constexpr int BM = 128;                     // rows of A per CTA
constexpr int BN = 256;                     // accumulator columns (rows of B per pair)
constexpr int BK = 64;                      // contraction elements per block: 128 bytes
constexpr int UMMA_K = 16;
constexpr int OP_BYTES = 128 * BK * 2;      // 16 KB: 128 rows of an operand
constexpr int MN_BLOCK = 64 * BK * 2;       // 8 KB: 64 columns x 64 contraction rows of an MN-major operand
// Stages of the ring: A and B, or A in two terms and B; 192 KB either way.
__host__ __device__ constexpr int stages(int parts) { return parts == 2 ? 4 : 6; }
constexpr int RING_BYTES = 192 * 1024;
static_assert(stages(1) * 2 * OP_BYTES == RING_BYTES && stages(2) * 3 * OP_BYTES == RING_BYTES, "ring");
constexpr int SMEM_BYTES = RING_BYTES + 1024 + 256;
constexpr int EPI_WARP0 = 4;
constexpr int EPI_GROUP = 4;                // epilogue warps of a region, one per TMEM lane quarter (two: 368 us against 350)
constexpr int THREADS = (EPI_WARP0 + 2 * EPI_GROUP) * 32;
// Row-tiles that share B's tiles in L2 before the next columns: backward 8 (4 and
// 16 within 1 % under the power cap); forward, so many that their rows of X are
// about 32 MB (16 at K=4096: 345 us against 351 for 8 and 367 for 4).
constexpr int GROUP_BACK = 8;
constexpr uint64_t GROUP_X_BYTES = 32ull << 20;
constexpr int MAX_SPLIT = 4;

constexpr uint32_t SITE_PRODUCER = 0x00070001u;
constexpr uint32_t SITE_MMA_FULL = 0x00070002u;
constexpr uint32_t SITE_MMA_TMEM = 0x00070003u;
constexpr uint32_t SITE_EPI = 0x00070004u;

struct Barriers {
    uint64_t full[6];
    uint64_t empty[6];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

// Tensor maps: forward X, Wg, Wu; backward also dG and dU with their remainders.
struct Maps {
    CUtensorMap x, wg, wu;
    CUtensorMap rows[2][2]; // [dG, dU][value, remainder] in boxes of 128 rows (dX)
    CUtensorMap cols[2][2]; // the same in boxes of 64 rows (dWg, dWu)
};

struct Params {
    int M, N, K;
    int tiles_dx, tiles_dw; // tiles of dX and of each of dWg, dWu (0: not computed)
    int tiles;              // in all
    int first;              // of them those with the longer contraction come first: dX's,
    int dw_first;           // or dWg's and dWu's
    int ratio;              // see nth_tile
    int whole_from;         // SPLIT: tiles from this one on are not split
    int group_m;            // forward: row-tiles per group
    void* out0;             // H, or dX
    void* out1;             // G (or null), or dWg
    void* out2;             // U (or null), or dWu
    DeviceStatus* status;
};

// One tile: what it is of, where, and how many 64-deep blocks it sums.
struct Tile {
    int kind;               // FWD, DX, DW
    int which;              // DW: 0 dWg, 1 dWu
    int mt, nt;
    int rows, cols;         // of the output
    int nk;
};

template <bool BACK>
__device__ __forceinline__ Tile find_tile(int t, const Params& p) {
    constexpr int TN = BACK ? BN : BN / 2;                      // output columns of a tile
    Tile r;
    if constexpr (!BACK) {
        r.kind = FWD; r.which = 0; r.rows = p.M; r.cols = p.N; r.nk = (p.K + BK - 1) / BK;
    } else {
        const bool head = t < p.first;
        if (!head) t -= p.first;
        if (head != (p.dw_first != 0)) {
            r.kind = DX; r.which = 0; r.rows = p.M; r.cols = p.K; r.nk = 2 * ((p.N + BK - 1) / BK);
        } else {
            r.kind = DW; r.which = t >= p.tiles_dw; r.rows = p.N; r.cols = p.K; r.nk = (p.M + BK - 1) / BK;
            if (r.which) t -= p.tiles_dw;
        }
    }
    const int tiles_m = (r.rows + 2 * BM - 1) / (2 * BM), tiles_n = (r.cols + TN - 1) / TN;
    const int group_m = BACK ? GROUP_BACK : p.group_m;
    const int group = group_m * tiles_n;
    const int g = t / group;
    const int first_m = g * group_m;
    const int gm = min(tiles_m - first_m, group_m);
    const int q = t - g * group;
    r.mt = first_m + q % gm;
    r.nt = q / gm;
    return r;
}

// The n-th tile of a pair (p.tiles or more: none).  Tiles go round the pairs; where
// the long ones leave some pairs one short, those take as many more of the short
// ones first (`ratio` = blocks of a long tile per block of a short one).
template <bool BACK>
__device__ __forceinline__ int nth_tile(int n, int pair, int pairs, const Params& p) {
    const int extra = BACK ? p.first % pairs : 0;             // pairs with one long tile more
    if (extra == 0 || p.first == p.tiles) return pair + n * pairs;
    const int mine = p.first / pairs + (pair < extra ? 1 : 0);
    if (n < mine) return pair + n * pairs;
    n -= mine;
    const int others = pairs - extra;
    if (pair >= extra) {
        if (n < p.ratio) return p.first + (pair - extra) + n * others;
        n -= p.ratio;
    }
    return p.first + others * p.ratio + pair + n * pairs;
}

// The one tile of pair `sub` in cluster `c` of a SPLIT launch: the cluster's own, of
// which it takes a part, or from p.whole_from on one for each pair (p.tiles or
// more: none).
__device__ __forceinline__ int cluster_tile(int c, int sub, int subs, const Params& p) {
    return c < p.whole_from ? c : p.whole_from + (c - p.whole_from) * subs + sub;
}

// Where pair `sub` of `subs` begins in a tile of nk blocks.  A tile of fewer
// blocks than pairs gives the first nk pairs one each and the others none.
__device__ __forceinline__ int part_begin(int nk, int sub, int subs) {
    const int n = min(subs, nk);
    return sub >= n ? nk : (int)((int64_t)nk * sub / n);
}

// 128 rows of an operand: K-major in one box, MN-major in two side by side.
// Coordinates are in bytes along x (the maps describe byte matrices).
template <bool MN>
__device__ __forceinline__ void load_operand(uint8_t* dst, const CUtensorMap* map, uint32_t bar, int row0, int k0) {
    if constexpr (MN) {
        tma_load_2d_pair(dst, map, bar, row0 * 2, k0);
        tma_load_2d_pair(dst + MN_BLOCK, map, bar, row0 * 2 + 128, k0);
    } else {
        tma_load_2d_pair(dst, map, bar, k0 * 2, row0);
    }
}

template <typename T>
__device__ __forceinline__ void store32(void* out, int row0, const Tile& tl, int n0, const float (&f)[32]) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = make_uint4(Pack<T>::two(f[8 * i], f[8 * i + 1]), Pack<T>::two(f[8 * i + 2], f[8 * i + 3]),
                          Pack<T>::two(f[8 * i + 4], f[8 * i + 5]), Pack<T>::two(f[8 * i + 6], f[8 * i + 7]));
    store_rows(static_cast<uint16_t*>(out), row0, tl.rows, n0, tl.cols, true, v);
}

// The results of 32 columns (forward: 32 outputs) of the warp's rows row0 + lane.
template <typename T, bool BACK, int ACT>
__device__ __forceinline__ void finish32(const Params& p, const Tile& tl, int row0, int n0, const uint32_t (&r0)[32],
                                         const uint32_t (&r1)[32]) {
    if (row0 >= tl.rows || n0 >= tl.cols) return;
    float f[32];
    if constexpr (BACK) {
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r0[i]);
        store32<T>(tl.kind == DX ? p.out0 : tl.which ? p.out2 : p.out1, row0, tl, n0, f);
    } else {
        if (p.out1) {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r0[i]);
            store32<T>(p.out1, row0, tl, n0, f);
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r1[i]);
            store32<T>(p.out2, row0, tl, n0, f);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = gated<ACT, true>(__uint_as_float(r0[i]), __uint_as_float(r1[i]));
        store32<T>(p.out0, row0, tl, n0, f);
    }
}

template <typename T, bool BACK, int ACT, bool SPLIT, int PARTS>   // PARTS: terms of dG and dU
__global__ void __launch_bounds__(THREADS, 1)
gated_kernel(const __grid_constant__ Maps maps, const Params p) {
    constexpr int TN = BACK ? BN : BN / 2;                  // output columns of a tile
    constexpr int STAGES = stages(PARTS), A_BYTES = PARTS * OP_BYTES;
    constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t IDESC = make_idesc(1, FMT, FMT, 2 * BM, BN);
    constexpr uint32_t A_MN = 1u << 15, B_MN = 1u << 16;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * A_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(smem + RING_BYTES);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);   // uniform, and known to be
    const int lane = threadIdx.x & 31;
    const uint32_t crank = cluster_rank();
    const uint32_t rank = crank & 1u, sub = crank >> 1;     // CTA of the pair, pair of the cluster
    const uint32_t leader_cta = crank & ~1u;
    const bool leader = rank == 0;
    const int subs = SPLIT ? (int)(cluster_size() >> 1) : 1;
    const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const int cluster = (int)blockIdx.x / (2 * subs);       // SPLIT: all that the pairs do is in here
    const bool parted = SPLIT && cluster < p.whole_from;    // and whether it is a part of a tile
    auto tile_at = [&](int n) {
        if constexpr (SPLIT) return n == 0 ? cluster_tile(cluster, (int)sub, subs, p) : p.tiles;
        else return nth_tile<BACK>(n, pair, pairs, p);
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(&bars->tmem_full[a], 1); mbar_init(&bars->tmem_empty[a], 2 * EPI_GROUP); }
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&maps.x);
        tma_prefetch_desc(&maps.wg);
        tma_prefetch_desc(&maps.wu);
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
        for (int n = 0, t; ok && (t = tile_at(n)) < p.tiles; ++n) {
            const Tile tl = find_tile<BACK>(t, p);
            const int i0 = parted ? part_begin(tl.nk, (int)sub, subs) : 0, i1 = parted ? part_begin(tl.nk, (int)sub + 1, subs) : tl.nk;
            const int m0 = tl.mt * 2 * BM + (int)rank * BM;
            const int nb = (p.N + BK - 1) / BK;
            for (int i = i0; i < i1; ++i) {
                if (!mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER)) { ok = false; break; }
                if (leader) mbar_arrive_expect_tx(&bars->full[stage], 2 * (A_BYTES + OP_BYTES));
                const uint32_t full = mapa_shared(smem_u32(&bars->full[stage]), leader_cta);
                uint8_t* da = sA + stage * A_BYTES;
                uint8_t* db = sB + stage * OP_BYTES;
                if constexpr (!BACK) {
                    load_operand<false>(da, &maps.x, full, m0, i * BK);
                    load_operand<false>(db, leader ? &maps.wg : &maps.wu, full, tl.nt * 128, i * BK);
                } else {
                    int j = i;
                    const CUtensorMap* b = &maps.x;
                    if (tl.kind == DX) {
                        const int seg = j >= nb;
                        if (seg) j -= nb;
                        b = seg ? &maps.wu : &maps.wg;
#pragma unroll
                        for (int q = 0; q < PARTS; ++q)
                            load_operand<false>(da + q * OP_BYTES, &maps.rows[seg][q], full, m0, j * BK);
                    } else {
#pragma unroll
                        for (int q = 0; q < PARTS; ++q)
                            load_operand<true>(da + q * OP_BYTES, &maps.cols[tl.which][q], full, m0, j * BK);
                    }
                    load_operand<true>(db, b, full, tl.nt * BN + (int)rank * 128, j * BK);
                }
                armed |= 1u << stage;
                armed_phase = (armed_phase & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        // the even CTA's last commits land here before this CTA's shared memory goes away
        for (int i = 0; i < STAGES && ok; ++i) {
            ok = mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, SITE_PRODUCER);
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok && leader) {
            // copies of both CTAs complete on these barriers: let them land
            for (int s = 0; s < STAGES; ++s)
                if (armed & (1u << s)) mbar_wait(&bars->full[s], (armed_phase >> s) & 1u, nullptr, nullptr, 0);
        }
    } else if (warp == 1 && leader) {
        // ------------------------------------------------------------ MMA issuer (even CTA)
        // The whole warp walks the blocks and one elected lane issues: descriptors
        // and barrier addresses stay in uniform registers.
        const uint32_t a_addr = smem_u32(sA), b_addr = smem_u32(sB);
        uint32_t stage = 0, phase = 0;
        bool ok = true, issued = false;
        int unit = 0;
        for (int n = 0, t; ok && (t = tile_at(n)) < p.tiles; ++n, ++unit) {
            const Tile tl = find_tile<BACK>(t, p);
            const int i0 = parted ? part_begin(tl.nk, (int)sub, subs) : 0, i1 = parted ? part_begin(tl.nk, (int)sub + 1, subs) : tl.nk;
            auto blocks = [&](auto a_major) {
                constexpr bool A_IS_MN = decltype(a_major)::value;
                const uint64_t a_desc = A_IS_MN ? make_sdesc_mnmajor_sw128(a_addr, MN_BLOCK) : make_sdesc_kmajor_sw128(a_addr);
                const uint64_t b_desc = BACK ? make_sdesc_mnmajor_sw128(b_addr, MN_BLOCK) : make_sdesc_kmajor_sw128(b_addr);
                // 16 contraction elements: 32 bytes of a K-major row, 16 rows of an MN-major tile
                constexpr uint32_t A_STEP = A_IS_MN ? UMMA_K * 128 >> 4 : UMMA_K * 2 >> 4;
                constexpr uint32_t B_STEP = BACK ? UMMA_K * 128 >> 4 : UMMA_K * 2 >> 4;
                constexpr uint32_t ID = IDESC | (A_IS_MN ? A_MN : 0u) | (BACK ? B_MN : 0u);
                const uint32_t region = unit & 1, use = unit >> 1;
                for (int i = i0; i < i1; ++i) {
                    if (!warp_wait(&bars->full[stage], phase, abort_flag, p.status, SITE_MMA_FULL)) return false;
                    if (i == i0 && !warp_wait(&bars->tmem_empty[region], (use & 1) ^ 1u, abort_flag, p.status, SITE_MMA_TMEM))
                        return false;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t ad = a_desc + stage * (A_BYTES >> 4), bd = b_desc + stage * (OP_BYTES >> 4);
#pragma unroll
                        for (int q = 0; q < PARTS; ++q)
#pragma unroll
                            for (int k = 0; k < BK / UMMA_K; ++k)
                                umma_f16_pair(tmem_base + region * BN, ad + q * (OP_BYTES >> 4) + k * A_STEP, bd + k * B_STEP,
                                              ID, i != i0 || (q | k) != 0 ? 1u : 0u);
                        umma_commit_both(&bars->empty[stage], sub);
                        if (i + 1 == i1) umma_commit_both(&bars->tmem_full[region], sub);
                    }
                    __syncwarp();
                    issued = true;
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
                return true;
            };
            if (BACK && tl.kind == DW) ok = blocks(std::true_type{});
            else ok = blocks(std::false_type{});
        }
        if (!ok && issued && elect_one()) {
            umma_commit_pair(mapa_shared(smem_u32(&bars->drain), crank));
            mbar_wait(&bars->drain, 0, nullptr, nullptr, 0);
        }
    } else if (warp >= EPI_WARP0) {
        // ------------------------------------------------------------ epilogue (both CTAs)
        auto release = [&](uint32_t region) {                     // the region may be overwritten
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_relaxed(mapa_shared(smem_u32(&bars->tmem_empty[region]), leader_cta));
        };
        // Tile n belongs to group n % 2; the pair's last tile to both, half of the columns
        // each (an only tile's epilogue is 7000 of 15000 clocks at 1000x512x512).
        const int group = (warp - EPI_WARP0) / EPI_GROUP;
        const int row = (warp & 3) * 32 + lane;
        for (int n = 0;; ++n) {
            const int t = tile_at(n);
            if (t >= p.tiles) break;
            const bool last = tile_at(n + 1) >= p.tiles;
            const uint32_t region = n & 1;
            if (!last && (int)region != group) continue;
            const Tile tl = find_tile<BACK>(t, p);
            const int m_warp = tl.mt * 2 * BM + (int)rank * BM + (warp & 3) * 32;
            if (parted && (int)sub >= tl.nk) break;               // no blocks, no part
            if (!warp_wait(&bars->tmem_full[region], (n >> 1) & 1, abort_flag, p.status, SITE_EPI)) break;
            tc_fence_after();
            const bool some = m_warp < tl.rows;                   // (no rows in this warp: nothing to read)
            const uint32_t t_row = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + region * BN;
            if (parted) {
                // this pair's part of the sums, column by column over the drained ring
                float* part = reinterpret_cast<float*>(smem) + row;
#pragma unroll 1
                for (int c = group * (BN / 2); some && c < (group + 1) * (BN / 2); c += 32) {
                    uint32_t r[32];
                    __syncwarp();
                    tmem_ld_32x32b_x32(t_row + c, r);
                    tmem_ld_wait_regs(r);
#pragma unroll
                    for (int i = 0; i < 32; ++i) part[(c + i) * BM] = __uint_as_float(r[i]);
                }
            } else {
                const int c_end = last ? (group + 1) * (TN / 2) : TN;
#pragma unroll 1
                for (int c = last ? group * (TN / 2) : 0; some && c < c_end; c += 32) {
                    uint32_t r0[32], r1[32];
                    __syncwarp();
                    tmem_ld_32x32b_x32(t_row + c, r0);
                    if constexpr (!BACK) tmem_ld_32x32b_x32(t_row + BN / 2 + c, r1);
                    tmem_ld_wait_regs(r0);
                    if constexpr (!BACK) tmem_ld_wait_regs(r1);
                    if (!last && c + 32 == TN) release(region);   // the warp's last columns are in registers
                    finish32<T, BACK, ACT>(p, tl, m_warp, tl.nt * TN + c, r0, r1);
                }
                if (!last && !some) release(region);
            }
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
    if constexpr (SPLIT) {
        // every CTA joins its share of the columns, 32 at a time, from the same CTA of each pair
        if (warp >= EPI_WARP0 && parted) {
            const Tile tl = find_tile<BACK>(cluster, p);
            const int row = (warp & 3) * 32 + lane;
            const int m_warp = tl.mt * 2 * BM + (int)rank * BM + (warp & 3) * 32;
            const uint32_t base = smem_u32(smem) + (uint32_t)row * 4;
            const int c_end = m_warp < tl.rows ? TN : 0;        // (no rows in this warp: nothing)
            for (int c = ((int)sub + subs * ((warp - EPI_WARP0) >> 2)) * 32; c < c_end; c += subs * (2 * EPI_GROUP / 4) * 32) {
                uint32_t r0[32] = {}, r1[32] = {};               // fp32 zeros
                for (int k = 0; k < min(subs, tl.nk); ++k) {
                    const uint32_t at = mapa_shared(base + (uint32_t)(c * BM) * 4, 2u * k + rank);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        r0[i] = __float_as_uint(__uint_as_float(r0[i]) + ld_cluster_f32(at + i * BM * 4));
                        if constexpr (!BACK)
                            r1[i] = __float_as_uint(__uint_as_float(r1[i]) + ld_cluster_f32(at + (BN / 2 + i) * BM * 4));
                    }
                }
                finish32<T, BACK, ACT>(p, tl, m_warp, tl.nt * TN + c, r0, r1);
            }
        }
        cluster_sync();                                           // nobody leaves while its part is being read
    }
}

// dG = dH * U * act'(G), dU = dH * act(G), eight elements per thread, in `parts`
// terms (the value rounded to T, and what that left out).  Five streams of
// 2 bytes per element: bound by memory (4096x8192 in 47 us, 7.1 TB/s).
template <typename T, int ACT, int PARTS>
__global__ void __launch_bounds__(256)
gate_backward_kernel(const uint4* dH, const uint4* G, const uint4* U,
                     uint4* D, uint64_t n8) {
    wait_previous_grid();
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n8) return;
    const uint4 vh = load_global(dH + i), vg = load_global(G + i), vu = load_global(U + i);
    const uint32_t h[4] = {vh.x, vh.y, vh.z, vh.w}, g[4] = {vg.x, vg.y, vg.z, vg.w}, u[4] = {vu.x, vu.y, vu.z, vu.w};
    uint32_t o[2][2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 fh = Pack<T>::unpack(h[j]), fg = Pack<T>::unpack(g[j]), fu = Pack<T>::unpack(u[j]);
        float a0, s0, a1, s1;
        gate_slope<ACT>(fg.x, a0, s0);
        gate_slope<ACT>(fg.y, a1, s1);
        const float d[2][2] = {{fh.x * fu.x * s0, fh.y * fu.y * s1}, {fh.x * a0, fh.y * a1}};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            o[w][0][j] = Pack<T>::two(d[w][0], d[w][1]);
            if constexpr (PARTS == 2) {
                const float2 r = Pack<T>::unpack(o[w][0][j]);
                // (a value past the type's range has no remainder: infinity stays infinity)
                o[w][1][j] = Pack<T>::two(isinf(r.x) ? 0.0f : d[w][0] - r.x, isinf(r.y) ? 0.0f : d[w][1] - r.y);
            }
        }
    }
    // D: dG, dU, then their remainders, n8 words each
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
            D[(uint64_t)(2 * q + w) * n8 + i] = make_uint4(o[w][q][0], o[w][q][1], o[w][q][2], o[w][q][3]);
}

// The byte matrix of a 2-byte tensor [rows, cols] in boxes of 128 bytes x box_rows.
static int make_map(CUtensorMap* map, const void* base, int rows, int cols, int box_rows) {
    return make_tmap_2d(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)cols * 2, (uint64_t)rows,
                        (uint64_t)cols * 2, 128, (uint32_t)box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Clusters of `ctas` CTAs that can be resident at once (they need free SMs of one
// GPC, so this can be below sm_count / ctas).  All forms of the kernel have the
// same block and shared-memory size, so `kernel` stands for all of them.
static int resident_clusters(void (*kernel)(Maps, Params), int ctas, int* out, const DeviceInfo* info) {
    static std::atomic<int> known[64][2 * MAX_SPLIT + 1];     // 0: not asked yet
    int dev = 0;
    QG_CUDA(cudaGetDevice(&dev));
    std::atomic<int>& res = known[dev & 63][ctas];
    if (!res) {
        QG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        cudaLaunchConfig_t lc = {};
        lc.gridDim = dim3(info->sm_count / ctas * ctas);
        lc.blockDim = dim3(THREADS);
        lc.dynamicSmemBytes = SMEM_BYTES;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {(unsigned)ctas, 1, 1};
        lc.attrs = at;
        lc.numAttrs = 1;
        int n = 0;
        QG_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &lc));
        res = n > 0 ? n : 1;
    }
    *out = res;
    return QG_OK;
}

template <typename T, bool BACK, int ACT, bool SPLIT, int PARTS>
static int launch_kernel(const Maps& maps, Params p, int subs, const DeviceInfo* info, cudaStream_t stream) {
    constexpr int TN = BACK ? BN : BN / 2;
    if constexpr (!BACK) p.tiles = ceil_div(p.M, 2 * BM) * ceil_div(p.N, TN);
    else {
        if (p.tiles_dx) p.tiles_dx = ceil_div(p.M, 2 * BM) * ceil_div(p.K, TN);
        if (p.tiles_dw) p.tiles_dw = ceil_div(p.N, 2 * BM) * ceil_div(p.K, TN);
        p.tiles = p.tiles_dx + 2 * p.tiles_dw;
        p.first = p.dw_first ? 2 * p.tiles_dw : p.tiles_dx;
    }
    auto kernel = gated_kernel<T, BACK, ACT, SPLIT, PARTS>;
    QG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
    int pairs = 0;
    if constexpr (SPLIT) {
        // (a backward pass splits all its tiles, or the long ones)
        p.whole_from = p.whole_from ? p.first : p.tiles;
        pairs = (p.whole_from + ceil_div(p.tiles - p.whole_from, subs)) * subs;
    }
    else {
        int rc = resident_clusters(kernel, 2, &pairs, info);
        if (rc) return rc;
        if (p.tiles < pairs) pairs = p.tiles;
    }
    QG_CUDA(launch_overlapped(kernel, dim3(2 * pairs), dim3(THREADS), SMEM_BYTES, stream, 2 * subs, maps, p));
    return QG_OK;
}

// Pairs per tile, of `units` tiles and `nk` blocks in the longest: 4 or 2 while all
// the clusters fit at once and the contraction is long enough.  Joining the parts
// costs about 4.5 us (128 KB per CTA over distributed shared memory), a block
// 0.3 us.  Forward (where use_rows leaves it: two pairs), split / whole:
// 512x2048x1280 (20 blocks) 12.5 / 11.0 us, 512x2048x2048 (32) 14.6 / 14.6,
// 256x4096x4096 (64) 20.6 / 24.1.  Backward: 256x768x512 (24) 13.4 / 12.7,
// 2000x256x1024 (32) 14.7 / 15.6, 512x960x1024 (30) 14.1 / 15.1.
constexpr int split_min_blocks(bool back) { return back ? 20 : 32; }
template <typename T, bool BACK, int ACT>
static int pick_split(int* out, int64_t units, int nk, const DeviceInfo* info) {
    *out = 1;
    for (int s = 2; s <= MAX_SPLIT && nk >= split_min_blocks(BACK); s *= 2) {
        int clusters = 0;
        const int rc = resident_clusters(gated_kernel<T, BACK, ACT, true, 1>, 2 * s, &clusters, info);
        if (rc) return rc;
        if (units <= clusters) *out = s;
    }
    return QG_OK;
}

template <typename T, bool BACK, int ACT, int PARTS = 1>
static int launch(const Maps& maps, Params p, int64_t units, int nk, const DeviceInfo* info, cudaStream_t stream) {
    int rc;
    if ((rc = device_status_ptr(&p.status))) return rc;
    int subs = 1;
    if ((rc = pick_split<T, BACK, ACT>(&subs, units, nk, info))) return rc;
    return subs > 1 ? launch_kernel<T, BACK, ACT, true, PARTS>(maps, p, subs, info, stream)
                    : launch_kernel<T, BACK, ACT, false, PARTS>(maps, p, 1, info, stream);
}

static int check_shape(const char* name, int M, int N, int K) {
    QG_CHECK_ARG(M > 0 && N > 0 && K > 0, "%s: empty shape %dx%dx%d", name, M, N, K);
    QG_CHECK_ARG(N % 8 == 0 && K % 8 == 0, "%s: N=%d and K=%d must be multiples of 8 (16-byte rows)", name, N, K);
    // x coordinates are bytes in 32 bits; tile counts fit too
    QG_CHECK_ARG(M <= (1 << 29) && N <= (1 << 29) && K <= (1 << 29), "%s: shape %dx%dx%d is too large", name, M, N, K);
    const int64_t m = ceil_div(M, 256), n = ceil_div(N, 128), k = ceil_div(K, 256);
    QG_CHECK_ARG(m * n <= (1 << 29) && m * k <= (1 << 29) && n * k <= (1 << 29), "%s: shape %dx%dx%d is too large", name, M, N, K);
    return QG_OK;
}

// Terms of dG and dU (see the head of this file).
static int grad_parts(int M, int N) { return (int64_t)M * N <= 65536 ? 2 : 1; }

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
    DeviceInfo* info = nullptr;
    if ((rc = current_device_info(&info))) return rc;
    if (use_rows(M, N, K, info->sm_count))
        return gated_rows(X, Wg, Wu, H, G, U, std::is_same<T, __half>::value, act, M, N, K, info->sm_count, stream);
    Maps maps;
    if ((rc = make_map(&maps.x, X, M, K, BM)) || (rc = make_map(&maps.wg, Wg, N, K, 128)) ||
        (rc = make_map(&maps.wu, Wu, N, K, 128)))
        return rc;
    for (int i = 0; i < 4; ++i) maps.rows[i >> 1][i & 1] = maps.cols[i >> 1][i & 1] = maps.x;   // not read
    const uint64_t group = GROUP_X_BYTES / ((uint64_t)2 * BM * (uint64_t)K * 2);
    const Params p{M, N, K, 0, 0, 0, 0, 0, 0, 0, (int)(group < 1 ? 1 : group > 64 ? 64 : group), H, G, U, nullptr};
    const int64_t units = (int64_t)ceil_div(M, 2 * BM) * ceil_div(N, BN / 2);
    return act == QG_ACT_SILU ? launch<T, false, QG_ACT_SILU>(maps, p, units, ceil_div(K, BK), info, stream)
                              : launch<T, false, QG_ACT_GELU_TANH>(maps, p, units, ceil_div(K, BK), info, stream);
}

// Whether dX goes to the kernel for few rows, in a launch apart from dWg's and dWu's:
// more rows only where its contraction is long enough to outweigh that, or where dX
// would have a launch of its own anyway.  All gradients, in one launch / with dX apart:
// 1x8192x4096 109 / 62 us, 16x8192x4096 78 / 61, 64x1024x4096 25.6 / 18.3, 64x512x512
// 15.0 / 12.2, 128x1024x512 13.5 / 13.1, 256x4096x1024 31.1 / 25.3, 512x8192x512 45.5 /
// 36.6; 256x1024x1024 14.5 / 16.2, 512x2048x512 17.8 / 20.5, 1024x512x512 11.4 / 17.6.
// In two launches of the pairs / with dX here: 256x1024x2048 21.6 / 16.7,
// 384x2048x1024 25.0 / 19.9, 768x4096x512 34.3 / 28.8.
static bool use_rows_dx(int M, int N, int K, bool apart_anyway, int sms) {
    return M <= 64 || (rows_split_dx(M, N, K, sms) >= 4 && (apart_anyway || M <= 10 * ceil_div(N, BK)));
}

// The products of the backward pass; rows_dx() launches dX by the kernel for few rows.
template <typename T, int PARTS, typename F>
static int products(const Maps& maps, const F& rows_dx, void* dX, void* dWg, void* dWu, int M, int N, int K,
                    const DeviceInfo* info, cudaStream_t stream) {
    int rc;
    const int nk_dx = 2 * ceil_div(N, BK), nk_dw = ceil_div(M, BK);
    const int64_t units_dx = (int64_t)ceil_div(M, 2 * BM) * ceil_div(K, BN);
    const int64_t units_dw = 2 * (int64_t)ceil_div(N, 2 * BM) * ceil_div(K, BN);
    auto dx_apart = [&] {
        const Params p{M, N, K, 0, 1, 0, 0, 1, 1, 0, 1, nullptr, dWg, dWu, nullptr};
        if (dX && (rc = rows_dx())) return rc;
        return dWg ? launch<T, true, QG_ACT_SILU, PARTS>(maps, p, units_dw, nk_dw, info, stream) : QG_OK;
    };
    if (use_rows_dx(M, N, K, false, info->sm_count)) return dx_apart();
    // One launch for the three: all tiles split; or the long ones, where they are few of
    // many blocks beside many of few (dX with few rows of X, dWg and dWu with many) and
    // all fit at once; or none split.  Where the long ones should be split and do not
    // fit beside the others, they go alone and the others follow.  (Decided for all
    // three, whichever are asked for: the same split, the same bits.)
    const bool dw_first = nk_dw > nk_dx;
    const int nk = dw_first ? nk_dw : nk_dx, nk_short = dw_first ? nk_dx : nk_dw;
    const int64_t units = dw_first ? units_dw : units_dx, units_short = dw_first ? units_dx : units_dw;
    const Params p{M, N, K, dX ? 1 : 0, dWg ? 1 : 0, 0, 0, dw_first, (nk + nk_short / 2) / nk_short, 0, 1, dX, dWg,
                   dWu, nullptr};
    int all = 1, alone = 1, beside = 1;
    if ((rc = pick_split<T, true, QG_ACT_SILU>(&all, units + units_short, nk, info)) ||
        (rc = pick_split<T, true, QG_ACT_SILU>(&alone, units, nk, info)))
        return rc;
    if (all == 1 && alone > 1 && nk > 2 * nk_short) {
        for (int s = 2; s <= MAX_SPLIT; s *= 2) {
            int clusters = 0;
            if ((rc = resident_clusters(gated_kernel<T, true, QG_ACT_SILU, true, 1>, 2 * s, &clusters, info))) return rc;
            if (units + (units_short + s - 1) / s <= clusters) beside = s;
        }
        Params q = p;
        if (beside > 1) {
            q.whole_from = 1;
            if ((rc = device_status_ptr(&q.status))) return rc;
            return launch_kernel<T, true, QG_ACT_SILU, true, PARTS>(maps, q, beside, info, stream);
        }
        if (!dw_first && use_rows_dx(M, N, K, true, info->sm_count)) return dx_apart();
        (dw_first ? q.tiles_dx : q.tiles_dw) = 0;
        if ((dw_first ? dWg : dX) && (rc = launch<T, true, QG_ACT_SILU, PARTS>(maps, q, units, nk, info, stream))) return rc;
        q = p;
        (dw_first ? q.tiles_dw : q.tiles_dx) = 0;
        if ((dw_first ? dX : dWg) && (rc = launch<T, true, QG_ACT_SILU, PARTS>(maps, q, units_short, nk_short, info, stream))) return rc;
        return QG_OK;
    }
    return launch<T, true, QG_ACT_SILU, PARTS>(maps, p, units + units_short, nk, info, stream);
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
    const int parts = grad_parts(M, N);
    const uint64_t one = (uint64_t)M * (uint64_t)N * 2;           // a multiple of 16
    QG_CHECK_ARG(workspace && workspace_bytes >= 2 * parts * one, "%s: workspace of %llu bytes, %llu needed", name,
                 (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)(2 * parts * one));
    QG_CHECK_ARG((((uintptr_t)dH | (uintptr_t)X | (uintptr_t)Wg | (uintptr_t)Wu | (uintptr_t)G | (uintptr_t)U |
                   (uintptr_t)dX | (uintptr_t)dWg | (uintptr_t)dWu | (uintptr_t)workspace) & 15) == 0,
                 "%s: operands, outputs and workspace must be 16-byte aligned", name);
    DeviceInfo* info = nullptr;
    if ((rc = current_device_info(&info))) return rc;
    const uint64_t n8 = one / 16, blocks = (n8 + 255) / 256;
    QG_CHECK_ARG(blocks <= INT32_MAX, "%s: shape %dx%d is too large", name, M, N);
    auto* vh = static_cast<const uint4*>(dH);
    auto* vg = static_cast<const uint4*>(G);
    auto* vu = static_cast<const uint4*>(U);
    const bool silu = act == QG_ACT_SILU;
    auto kernel = parts == 2 ? (silu ? gate_backward_kernel<T, QG_ACT_SILU, 2> : gate_backward_kernel<T, QG_ACT_GELU_TANH, 2>)
                             : (silu ? gate_backward_kernel<T, QG_ACT_SILU, 1> : gate_backward_kernel<T, QG_ACT_GELU_TANH, 1>);
    QG_CUDA(launch_overlapped(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, 1, vh, vg, vu,
                              static_cast<uint4*>(workspace), n8));
    auto rows_dx = [&] {
        const void* d[4] = {};
        for (int i = 0; i < 2 * parts; ++i) d[i] = static_cast<const uint8_t*>(workspace) + i * one;
        return gated_rows_dx(d, Wg, Wu, dX, std::is_same<T, __half>::value, M, N, K, info->sm_count, stream);
    };
    const bool no_dx = use_rows_dx(M, N, K, false, info->sm_count);             // (its operands' maps are not read)
    Maps maps;
    if ((rc = make_map(&maps.x, X, M, K, BK))) return rc;
    for (int w = 0; w < 2; ++w)
        for (int q = 0; q < 2; ++q) {
            void* d = static_cast<uint8_t*>(workspace) + (2 * q + w) * one;
            // (the second term of one is not read)
            if (q >= parts) maps.cols[w][q] = maps.cols[w][0];
            else if ((rc = make_map(&maps.cols[w][q], d, M, N, BK))) return rc;
            if (q >= parts || no_dx) maps.rows[w][q] = maps.cols[w][q];
            else if ((rc = make_map(&maps.rows[w][q], d, M, N, BM))) return rc;
        }
    maps.wg = maps.wu = maps.x;
    if (!no_dx && ((rc = make_map(&maps.wg, Wg, N, K, BK)) || (rc = make_map(&maps.wu, Wu, N, K, BK)))) return rc;
    return parts == 2 ? products<T, 2>(maps, rows_dx, dX, dWg, dWu, M, N, K, info, stream)
                      : products<T, 1>(maps, rows_dx, dX, dWg, dWu, M, N, K, info, stream);
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
    *bytes = 4ull * (uint64_t)qg::ffn::grad_parts(M, N) * (uint64_t)M * (uint64_t)N;
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
