// qg_quant_mxfp4.cu -- a tensor into MXFP4 (qg_mxfp4.cuh) and back.
//
// Both directions are streams: quantisation reads M K values and writes
// M K (1/2 + 1/32) bytes, so the memory system bounds them.  A warp takes 256
// consecutive columns of ROWS rows: a lane holds eight of them (one 16-byte
// load of a 2-byte type), the maximum of a block is two shuffles over its four
// lanes, the lane's eight codes are one 4-byte store and a row's four scales of
// an atom are one 4-byte store.  The ROWS loads of a lane are issued before the
// first use.
#include "qg_common.cuh"
#include "qg_formats.cuh"
#include "qg_launch.cuh"
#include "qg_mxfp4.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace qg {
namespace mx {

constexpr int SEG = 256;        // columns of a warp
constexpr int ROWS = 4;         // rows of a warp
constexpr int THREADS = 256;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// The lane's eight values; `n` of them exist, the others are zero.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* src, int n, float (&v)[8]) {
    if (VEC && n == 8) {
        constexpr int W = 8 * sizeof(T) / 16;
        uint4 raw[W];
#pragma unroll
        for (int i = 0; i < W; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
        const T* t = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32<T>(src[i]) : 0.0f;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS)
quant_kernel(const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ Q, uint8_t* __restrict__ SF, int M, int K) {
    const int lane = threadIdx.x & 31;
    const int kp = (K + BLOCK - 1) / BLOCK * BLOCK;          // columns that have codes
    const int kchunks = (K + ATOM_K - 1) / ATOM_K;
    const int segs = (kchunks * ATOM_K + SEG - 1) / SEG;
    const int row_groups = (M + 127) / 128 * (128 / ROWS);   // the rows that pad the last atom get zero scales
    const uint64_t units = (uint64_t)segs * (uint64_t)row_groups;
    const uint64_t step = (uint64_t)gridDim.x * (THREADS / 32);
    wait_previous_grid();
    for (uint64_t u = (uint64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); u < units; u += step) {
        const int rg = (int)(u / (uint32_t)segs);
        const int k0 = (int)(u - (uint64_t)rg * (uint32_t)segs) * SEG + lane * 8;
        const int r0 = rg * ROWS;
        const int n = min(8, max(0, K - k0));
        float v[ROWS][8];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            load8<T, VEC>(X + (int64_t)(r0 + i) * ldx + k0, r0 + i < M ? n : 0, v[i]);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            uint32_t amax = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const uint32_t s = scale_byte(amax);
            const float inv = inv_scale(s == 255 ? 0 : s);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= inv;
            const uint32_t w = s == 255 ? 0u : pack8(v[i]);
            if (r0 + i < M && k0 < kp)
                *reinterpret_cast<uint32_t*>(Q + (size_t)(r0 + i) * (kp / 2) + k0 / 2) = w;
            // lanes 0, 4, 8, 12 (16, 20, 24, 28) hold the four scales of one atom row
            const uint32_t pair = s | __shfl_down_sync(0xffffffffu, s, 4) << 8;
            const uint32_t four = pair | __shfl_down_sync(0xffffffffu, pair, 8) << 16;
            if ((lane & 15) == 0 && k0 / ATOM_K < kchunks)
                *reinterpret_cast<uint32_t*>(SF + sf_offset(r0 + i, k0 / BLOCK, kchunks)) = four;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
dequant_kernel(const uint8_t* __restrict__ Q, const uint8_t* __restrict__ SF, T* __restrict__ Y, int M, int K) {
    const int words = K / 8;                                   // 4-byte code words of a row
    const int kchunks = (K + ATOM_K - 1) / ATOM_K;
    const uint64_t total = (uint64_t)M * (uint32_t)words;
    const uint64_t step = (uint64_t)gridDim.x * THREADS;
    wait_previous_grid();
    for (uint64_t i = (uint64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += step) {
        const int r = (int)(i / (uint32_t)words);
        const int c = (int)(i - (uint64_t)r * (uint32_t)words);
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(Q) + i);
        const float s = scale_value(__ldg(SF + sf_offset(r, c >> 2, kchunks)));
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = code_value(w >> (4 * j)) * s;
        if constexpr (sizeof(T) == 4) {
            float4* d = reinterpret_cast<float4*>(Y + i * 8);
            d[0] = make_float4(f[0], f[1], f[2], f[3]);
            d[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // exact: two significant bits, the exponents of fp32
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                o[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(Y + i * 8) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

static int grid_for(uint64_t blocks, const DeviceInfo* info) {
    const uint64_t most = (uint64_t)info->sm_count * 8;         // 8 CTAs of 256 threads fill an SM
    return (int)(blocks < most ? (blocks ? blocks : 1) : most);
}

template <typename T>
static int launch_quant(const void* X, int64_t ldx, void* Q, void* SF, int M, int K, cudaStream_t s) {
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
    const int segs = ((K + ATOM_K - 1) / ATOM_K * ATOM_K + SEG - 1) / SEG;
    const uint64_t units = (uint64_t)segs * (uint64_t)((M + 127) / 128 * (128 / ROWS));
    const int grid = grid_for((units + THREADS / 32 - 1) / (THREADS / 32), info);
    const bool vec = ((uintptr_t)X & 15) == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0;
    const T* x = static_cast<const T*>(X);
    uint8_t* q = static_cast<uint8_t*>(Q);
    uint8_t* sf = static_cast<uint8_t*>(SF);
    QG_CUDA(launch_overlapped(vec ? quant_kernel<T, true> : quant_kernel<T, false>, dim3(grid), dim3(THREADS), 0, s, 1, x,
                              ldx, q, sf, M, K));
    return QG_OK;
}

} // namespace mx

uint64_t mxfp4_sf_bytes(int rows, int K) {
    return (uint64_t)((rows + 127) / 128) * (uint64_t)((K + mx::ATOM_K - 1) / mx::ATOM_K) * mx::ATOM_BYTES;
}

int quant_mxfp4(const void* X, int in_type, int64_t ldx, void* Q, void* SF, int M, int K, cudaStream_t s) {
    QG_CHECK_ARG(X && Q && SF, "qg_quant_mxfp4: null operand or output");
    QG_CHECK_ARG(M > 0 && K > 0, "qg_quant_mxfp4: empty shape %dx%d", M, K);
    QG_CHECK_ARG(M <= INT32_MAX - 127 && K <= INT32_MAX - 511, "qg_quant_mxfp4: shape %dx%d is too large", M, K);
    QG_CHECK_ARG(ldx >= K || M == 1, "qg_quant_mxfp4: row stride %lld below K=%d", (long long)ldx, K);
    QG_CHECK_ARG(((uintptr_t)Q & 15) == 0 && ((uintptr_t)SF & 15) == 0,
                 "qg_quant_mxfp4: codes and scales must be 16-byte aligned");
    const int esz = in_type == QG_OUT_F32 ? 4 : 2;
    QG_CHECK_ARG((uintptr_t)X % esz == 0, "qg_quant_mxfp4: X is not aligned to its element");
    switch (in_type) {
        case QG_OUT_BF16: return mx::launch_quant<__nv_bfloat16>(X, ldx, Q, SF, M, K, s);
        case QG_OUT_F16: return mx::launch_quant<__half>(X, ldx, Q, SF, M, K, s);
        case QG_OUT_F32: return mx::launch_quant<float>(X, ldx, Q, SF, M, K, s);
        default: set_error("qg_quant_mxfp4: in_type %d (bf16, f16 or f32)", in_type); return QG_ERR_ARG;
    }
}

int dequant_mxfp4(const void* Q, const void* SF, void* Y, int out_type, int M, int K, cudaStream_t s) {
    QG_CHECK_ARG(Q && SF && Y, "qg_dequant_mxfp4: null operand or output");
    QG_CHECK_ARG(M > 0 && K > 0, "qg_dequant_mxfp4: empty shape %dx%d", M, K);
    QG_CHECK_ARG(K % 32 == 0, "qg_dequant_mxfp4: K=%d must be a multiple of 32", K);
    QG_CHECK_ARG(((uintptr_t)Q & 15) == 0 && ((uintptr_t)SF & 15) == 0 && ((uintptr_t)Y & 15) == 0,
                 "qg_dequant_mxfp4: codes, scales and output must be 16-byte aligned");
    QG_CHECK_ARG(out_type == QG_OUT_BF16 || out_type == QG_OUT_F32, "qg_dequant_mxfp4: out_type %d (bf16 or f32)",
                 out_type);
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
    const int grid = mx::grid_for(((uint64_t)M * (uint64_t)(K / 8) + mx::THREADS - 1) / mx::THREADS, info);
    const uint8_t* q = static_cast<const uint8_t*>(Q);
    const uint8_t* sf = static_cast<const uint8_t*>(SF);
    if (out_type == QG_OUT_F32)
        QG_CUDA(launch_overlapped(mx::dequant_kernel<float>, dim3(grid), dim3(mx::THREADS), 0, s, 1, q, sf,
                                  static_cast<float*>(Y), M, K));
    else
        QG_CUDA(launch_overlapped(mx::dequant_kernel<__nv_bfloat16>, dim3(grid), dim3(mx::THREADS), 0, s, 1, q, sf,
                                  static_cast<__nv_bfloat16*>(Y), M, K));
    return QG_OK;
}

} // namespace qg

extern "C" int qg_mxfp4_sf_bytes(int rows, int K, uint64_t* bytes) {
    QG_CHECK_ARG(bytes && rows > 0 && K > 0, "qg_mxfp4_sf_bytes: bad argument");
    *bytes = qg::mxfp4_sf_bytes(rows, K);
    return QG_OK;
}

extern "C" int qg_quant_mxfp4(const void* X, int in_type, int64_t ldx, void* Q, void* SF, int M, int K, void* stream) {
    return qg::quant_mxfp4(X, in_type, ldx, Q, SF, M, K, static_cast<cudaStream_t>(stream));
}

extern "C" int qg_dequant_mxfp4(const void* Q, const void* SF, void* Y, int out_type, int M, int K, void* stream) {
    return qg::dequant_mxfp4(Q, SF, Y, out_type, M, K, static_cast<cudaStream_t>(stream));
}
