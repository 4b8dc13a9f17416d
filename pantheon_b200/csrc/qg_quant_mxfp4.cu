// qg_quant_mxfp4.cu -- a tensor into MXFP4 (qg_mxfp4.cuh) and back.
//
// Both directions are streams: quantisation reads M K values and writes
// M K (1/2 + 1/32) bytes, so the memory system bounds them, if the arithmetic
// stays near six instructions per value.  A lane holds 32 bytes of a row (sixteen
// 2-byte values or eight fp32), a warp 1 KB of each of ROWS rows; all loads of a
// lane are issued before the first use.  Magnitudes are compared as integers of
// their own type (two per instruction for 2-byte types), a block's maximum is one
// or two shuffles, scaling by a power of two is exact, and the conversion to codes
// is the hardware's.  Measured: 28672x8192 bf16 to codes 85.6 us (6.95 TB/s of reads
// and writes, 1.06 of the measured copy bandwidth), back to bf16 90 us (6.6 TB/s);
// 28672x4096 fp32 76 us (7.0 TB/s); rows off 16-byte boundaries, read as aligned words
// and shifted, 16384x8192 bf16 66 us (5.1 TB/s; value by value it was 104 us).
#include "qg_common.cuh"
#include "qg_formats.cuh"
#include "qg_launch.cuh"
#include "qg_mxfp4.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace qg {
namespace mx {

constexpr int SEG = 256;        // columns of a warp (dequantisation)
constexpr int ROWS = 4;         // rows of a warp
constexpr int ROWS_OFF = 2;     // rows of a warp off 16-byte boundaries (half as many again words per row)
constexpr int THREADS = 256;

// A lane's 32 bytes of a row.
template <typename T>
struct Raw {
    static constexpr int N = 32 / sizeof(T);        // values
    uint32_t w[8];
};

// The aligned 16-byte words around them: two, or three where the row is off a
// 16-byte boundary.
template <bool VEC>
struct Words {
    uint32_t w[VEC ? 8 : 12];
};

// Loads a lane's words; `n` of its values exist.  Off the boundary the words reach
// up to 14 bytes before them and 16 behind, between rows too; that is memory of the
// tensor as long as they lie in [begin, end), its first and last byte; otherwise (its corners, and
// rows that end within the lane) the values are loaded one by one, in place.
template <typename T, bool VEC>
__device__ __forceinline__ void load(const T* src, int n, uintptr_t begin, uintptr_t end, Words<VEC>& v) {
    constexpr int N = Raw<T>::N;
    const uintptr_t at = reinterpret_cast<uintptr_t>(src), base = at & ~(uintptr_t)15;
    const bool whole = n == N && (VEC || (base >= begin && base + 48 <= end));
    if (whole) {
#pragma unroll
        for (int i = 0; i < (VEC ? 2 : 3); ++i) {
            const uint4 q = load_global(reinterpret_cast<const uint4*>(base) + i);
            v.w[4 * i] = q.x; v.w[4 * i + 1] = q.y; v.w[4 * i + 2] = q.z; v.w[4 * i + 3] = q.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < (VEC ? 8 : 12); ++i) v.w[i] = 0;
    // as aligned words would hold them: value j at byte (at % 16) + j * sizeof(T)
    const int off = VEC ? 0 : (int)(at & 15);
#pragma unroll
    for (int i = 0; i < (VEC ? 8 : 12); ++i) {
        if constexpr (sizeof(T) == 4) {
            const int j = i - off / 4;
            if (j >= 0 && j < n) v.w[i] = load_global(reinterpret_cast<const uint32_t*>(src) + j);
        } else {
            const int j = 2 * i - off / 2;
            const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
            if (j >= 0 && j < n) v.w[i] = load_global(h + j);
            if (j + 1 >= 0 && j + 1 < n) v.w[i] |= load_global(h + j + 1) << 16;
        }
    }
}

// The lane's bytes out of its words (the offset is the same for the whole warp: a
// lane is 32 bytes).
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> align(const Words<VEC>& v, const T* src) {
    Raw<T> r;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = v.w[i];
    } else {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15);
        uint32_t t[10];
#pragma unroll
        for (int i = 0; i < 10; ++i) t[i] = (off & 8) ? v.w[i + 2] : v.w[i];
#pragma unroll
        for (int i = 0; i < 9; ++i) t[i] = (off & 4) ? t[i + 1] : t[i];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) r.w[i] = t[i];
        } else {
            const uint32_t shift = (off & 2) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) r.w[i] = __funnelshift_r(t[i], t[i + 1], shift);
        }
    }
    return r;
}

// Bits of the largest magnitude as its own type's integer: magnitudes of one type
// order as integers, NaN above infinity above the rest.
template <typename T>
__device__ __forceinline__ uint32_t max_bits(const Raw<T>& v) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        if constexpr (sizeof(T) == 4) m = __vimax3_u32(m, v.w[i] & 0x7FFFFFFFu, v.w[i + 1] & 0x7FFFFFFFu);
        else m = __vimax3_u16x2(m, v.w[i] & 0x7FFF7FFFu, v.w[i + 1] & 0x7FFF7FFFu);
    }
    return sizeof(T) == 4 ? m : max(m & 0xFFFFu, m >> 16);
}
template <typename T> __device__ __forceinline__ uint32_t f32_bits(uint32_t m);
template <> __device__ __forceinline__ uint32_t f32_bits<float>(uint32_t m) { return m; }
template <> __device__ __forceinline__ uint32_t f32_bits<__nv_bfloat16>(uint32_t m) { return m << 16; }
template <> __device__ __forceinline__ uint32_t f32_bits<__half>(uint32_t m) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}

// Value i of the lane.
template <typename T>
__device__ __forceinline__ float value(const Raw<T>& v, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v.w[i]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __uint_as_float((i & 1) ? v.w[i / 2] & 0xFFFF0000u : v.w[i / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short)((i & 1) ? v.w[i / 2] >> 16 : v.w[i / 2] & 0xFFFFu)));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS)
quant_kernel(const T* X, int64_t ldx, uint8_t* Q, uint8_t* SF, int M, int K) {
    constexpr int N = Raw<T>::N;                              // 16 or 8 values, 2 or 4 lanes per block
    const int lane = threadIdx.x & 31;
    const int kp = (K + BLOCK - 1) / BLOCK * BLOCK;          // columns that have codes
    const int kchunks = (K + ATOM_K - 1) / ATOM_K;
    const int segs = (kchunks * ATOM_K + 32 * N - 1) / (32 * N);
    constexpr int R = VEC ? ROWS : ROWS_OFF;
    const int row_groups = (M + 127) / 128 * (128 / R);      // the rows that pad the last atom get zero scales
    const uint64_t units = (uint64_t)segs * (uint64_t)row_groups;
    wait_previous_grid();
    const uint64_t u = (uint64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    if (u >= units) return;
    const int rg = (int)(u / (uint32_t)segs);
    const int k0 = (int)(u - (uint64_t)rg * (uint32_t)segs) * (32 * N) + lane * N;
    const int r0 = rg * R;
    const int n = min(N, max(0, K - k0));
    const uintptr_t begin = reinterpret_cast<uintptr_t>(X);
    const uintptr_t end = reinterpret_cast<uintptr_t>(X + (int64_t)(M - 1) * ldx + K);
    Words<VEC> words[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        load<T, VEC>(X + (int64_t)(r0 + i) * ldx + k0, r0 + i < M ? n : 0, begin, end, words[i]);
    uint8_t* q = Q + (size_t)r0 * (kp / 2) + k0 / 2;
    // the rows of a unit follow one another in their atom, 16 bytes apart
    uint8_t* sf = SF + sf_offset(r0, k0 / BLOCK, kchunks);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const Raw<T> v = align<T, VEC>(words[i], X + (int64_t)(r0 + i) * ldx + k0);
        uint32_t m = max_bits(v);
#pragma unroll
        for (int o = 1; o < BLOCK / N; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t s = scale_byte(f32_bits<T>(m));
        const float inv = inv_scale(s == 255 ? 0 : s);
        uint32_t w[N / 8];
#pragma unroll
        for (int g = 0; g < N / 8; ++g) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = value(v, 8 * g + j) * inv;
            w[g] = s == 255 ? 0u : pack8(f);
        }
        if (r0 + i < M && k0 < kp) {
            if constexpr (N == 16) *reinterpret_cast<uint2*>(q + (size_t)i * (kp / 2)) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(q + (size_t)i * (kp / 2)) = w[0];
        }
        // a row's four scales of an atom lie BLOCK / N lanes apart
        const uint32_t pair = s | __shfl_down_sync(0xffffffffu, s, BLOCK / N) << 8;
        const uint32_t four = pair | __shfl_down_sync(0xffffffffu, pair, 2 * BLOCK / N) << 16;
        if ((lane & (ATOM_K / N - 1)) == 0 && k0 < kchunks * ATOM_K) *reinterpret_cast<uint32_t*>(sf + 16 * i) = four;
    }
}

// Two codes to two fp32 values, exactly (through fp16).
__device__ __forceinline__ float2 unpack2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t}"
        : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The reverse, in the same shape: a lane's four bytes of a row are eight values.
template <typename T>
__global__ void __launch_bounds__(THREADS)
dequant_kernel(const uint8_t* Q, const uint8_t* SF, T* Y, int M, int K) {
    const int lane = threadIdx.x & 31;
    const int kchunks = (K + ATOM_K - 1) / ATOM_K;
    const int segs = (K + SEG - 1) / SEG;
    const uint64_t units = (uint64_t)segs * (uint64_t)((M + ROWS - 1) / ROWS);
    wait_previous_grid();
    const uint64_t u = (uint64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    if (u >= units) return;
    const int rg = (int)(u / (uint32_t)segs);
    const int k0 = (int)(u - (uint64_t)rg * (uint32_t)segs) * SEG + lane * 8;
    const int r0 = rg * ROWS;
    if (k0 >= K) return;
    uint32_t w[ROWS], s[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i < M ? r0 + i : M - 1;
        w[i] = load_global(reinterpret_cast<const uint32_t*>(Q + (size_t)r * (K / 2) + k0 / 2));
        s[i] = load_global(SF + sf_offset(r, k0 / BLOCK, kchunks));
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (r0 + i >= M) break;
        const float sc = scale_value(s[i]);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = unpack2(w[i] >> (8 * j));
            f[2 * j] = v.x * sc;
            f[2 * j + 1] = v.y * sc;
        }
        T* dst = Y + (size_t)(r0 + i) * K + k0;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // exact: two significant bits, the exponents of fp32
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                o[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// One warp per unit: short-lived CTAs keep every SM's queue of loads full to the
// end (a resident grid that walked the units took 391 us for 28672x8192 there and
// back).
static int grid_for(uint64_t units, const char* name, unsigned* grid) {
    const uint64_t blocks = (units + THREADS / 32 - 1) / (THREADS / 32);
    QG_CHECK_ARG(blocks <= INT32_MAX, "%s: tensor is too large", name);
    *grid = (unsigned)blocks;
    return QG_OK;
}

template <typename T>
static int launch_quant(const void* X, int64_t ldx, void* Q, void* SF, int M, int K, cudaStream_t s) {
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
    const int width = 32 * Raw<T>::N;
    const int segs = ((K + ATOM_K - 1) / ATOM_K * ATOM_K + width - 1) / width;
    const bool vec = ((uintptr_t)X & 15) == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0;
    const uint64_t units = (uint64_t)segs * (uint64_t)((M + 127) / 128 * (128 / (vec ? ROWS : ROWS_OFF)));
    unsigned grid = 0;
    if ((rc = grid_for(units, "qg_quant_mxfp4", &grid))) return rc;
    const T* x = static_cast<const T*>(X);
    uint8_t* q = static_cast<uint8_t*>(Q);
    uint8_t* sf = static_cast<uint8_t*>(SF);
    QG_CUDA(launch_overlapped(vec ? quant_kernel<T, true> : quant_kernel<T, false>, dim3(grid), dim3(THREADS), 0, s, 1, x,
                              ldx, q, sf, M, K));
    return QG_OK;
}

} // namespace mx

uint64_t mxfp4_sf_bytes(int rows, int K) {
    return ((uint64_t)rows + 127) / 128 * (((uint64_t)K + mx::ATOM_K - 1) / mx::ATOM_K) * mx::ATOM_BYTES;
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
    QG_CHECK_ARG(M <= INT32_MAX - 127 && K <= INT32_MAX - 511, "qg_dequant_mxfp4: shape %dx%d is too large", M, K);
    QG_CHECK_ARG(((uintptr_t)Q & 15) == 0 && ((uintptr_t)SF & 15) == 0 && ((uintptr_t)Y & 15) == 0,
                 "qg_dequant_mxfp4: codes, scales and output must be 16-byte aligned");
    QG_CHECK_ARG(out_type == QG_OUT_BF16 || out_type == QG_OUT_F32, "qg_dequant_mxfp4: out_type %d (bf16 or f32)",
                 out_type);
    DeviceInfo* info = nullptr;
    int rc = current_device_info(&info);
    if (rc) return rc;
    unsigned grid = 0;
    if ((rc = mx::grid_for((uint64_t)((K + mx::SEG - 1) / mx::SEG) * (uint64_t)((M + mx::ROWS - 1) / mx::ROWS),
                           "qg_dequant_mxfp4", &grid)))
        return rc;
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
