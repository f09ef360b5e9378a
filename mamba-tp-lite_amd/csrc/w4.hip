// Weights in 4-bit codes with group scales (gfx950): products with a few rows of x, and the matrix itself.
//   w[n, k] = s[n, k / G] (q[n, k] - z[n, k / G]),  q, z in 0..15 (z = 8 where none are given),  G = 32, 64 or 128
//   y[m, n] = bias[n] + sum_k x[m, k] w[n, k],      m < M <= 64
//
// Layout ("tiles", made once by ops.pack_w4): 16 rows x 128 columns of W are 1 KiB in the order in which a wavefront
// reads them, so one 16-byte load per lane takes a whole tile as one contiguous kilobyte.  Lane l = r + 16 j holds of
// row r, in its i-th word, the 8 codes of columns 32 i + 8 j + e; code e sits in nibble 4 (e & 1) + e / 2, so a shift
// and one and-or leave two neighbouring codes in the halves of a register.  Scales and zeros: [tiles, blocks, 16, 128/G].
// Rows and columns past N and K are there with scale 0.

#include "common.h"

namespace mtl {
namespace {

constexpr int kTileRows = 16, kBlockK = 128;

struct W4Args {
    const void* x;
    const uint8_t* codes;
    const void* scales;
    const uint8_t* zeros;
    const void* bias;
    void* y;
    int64_t ldx, ldy;
    int M, N, K, KB;           // KB: 128-column blocks of a row
};

// the code of column 32 i + 8 j + e in word w
__device__ __forceinline__ uint32_t code_of(uint32_t w, int e) { return (w >> (16 * (e & 1) + 4 * (e >> 1))) & 15u; }

template <typename S> __device__ __forceinline__ float scale_at(const void* p, int64_t i) {
    if constexpr (sizeof(S) == 2) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}

// One workgroup per 16 rows of W; wavefront w takes every 4th block of columns.  Each weight is made in fp32 as the
// matrix form rounds it, so an infinity or NaN in x meets it as it would meet the matrix.
template <typename T, typename S, int G, bool Z>
__global__ void __launch_bounds__(256) linear_w4_kernel(const W4Args a) {
    constexpr int NG = kBlockK / G;
    __shared__ float s_part[4][kTileRows];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, j = lane >> 4;
    const int64_t t = blockIdx.x;
    for (int m = 0; m < a.M; ++m) {
        const T* x = static_cast<const T*>(a.x) + m * a.ldx;
        float acc = 0.f;
        for (int kb = wave; kb < a.KB; kb += 4) {
            const uint4 w = reinterpret_cast<const uint4*>(a.codes)[(t * a.KB + kb) * 64 + lane];
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t at = ((t * a.KB + kb) * kTileRows + r) * NG + 32 * i / G;
                const float s = scale_at<S>(a.scales, at);
                const float z = Z ? (float)a.zeros[at] : 8.f;
                const int k0 = kb * kBlockK + 32 * i + 8 * j;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k0 + e < a.K) acc = fmaf(Act<T>::load(x + k0 + e), s * ((float)code_of(ws[i], e) - z), acc);
            }
        }
        acc += __shfl_xor(acc, 16);
        acc += __shfl_xor(acc, 32);
        if (lane < 16) s_part[wave][lane] = acc;
        __syncthreads();
        const int n = (int)t * kTileRows + threadIdx.x;
        if (threadIdx.x < kTileRows && n < a.N) {
            float v = (s_part[0][threadIdx.x] + s_part[1][threadIdx.x]) + (s_part[2][threadIdx.x] + s_part[3][threadIdx.x]);
            if (a.bias) v += Act<T>::load(static_cast<const T*>(a.bias) + n);
            Act<T>::store(static_cast<T*>(a.y) + m * a.ldy + n, v);
        }
        __syncthreads();
    }
}

// One wavefront per tile of 16 rows x 128 columns.
template <typename T, typename S, int G, bool Z>
__global__ void __launch_bounds__(256) dequantize_w4_kernel(const W4Args a) {
    constexpr int NG = kBlockK / G;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int64_t t = blockIdx.y + (int64_t)blockIdx.z * 65535;
    const int kb = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t n = t * kTileRows + r;
    if (kb >= a.KB || n >= a.N) return;
    const uint4 w = reinterpret_cast<const uint4*>(a.codes)[(t * a.KB + kb) * 64 + lane];
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    T* out = static_cast<T*>(a.y) + n * a.ldy;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t at = ((t * a.KB + kb) * kTileRows + r) * NG + 32 * i / G;
        const float s = scale_at<S>(a.scales, at);
        const float z = Z ? (float)a.zeros[at] : 8.f;
        const int k0 = kb * kBlockK + 32 * i + 8 * j;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k0 + e < a.K) Act<T>::store(out + k0 + e, s * ((float)code_of(ws[i], e) - z));
    }
}

// (T, S, G, Z) of a call
#define MTL_W4_G(KERNEL, T, S, Z, ...)                                             \
    switch (group) {                                                               \
        case 32: hipLaunchKernelGGL((KERNEL<T, S, 32, Z>), __VA_ARGS__); break;    \
        case 64: hipLaunchKernelGGL((KERNEL<T, S, 64, Z>), __VA_ARGS__); break;    \
        default: hipLaunchKernelGGL((KERNEL<T, S, 128, Z>), __VA_ARGS__); break;   \
    }
#define MTL_W4_Z(KERNEL, T, S, ...)                        \
    if (a.zeros) { MTL_W4_G(KERNEL, T, S, true, __VA_ARGS__) } else { MTL_W4_G(KERNEL, T, S, false, __VA_ARGS__) }
#define MTL_W4(KERNEL, ...)                                                                                     \
    if (dtype == MTL_F32) {                                                                                     \
        if (scale_dtype == MTL_F32) { MTL_W4_Z(KERNEL, float, float, __VA_ARGS__) }                             \
        else { MTL_W4_Z(KERNEL, float, uint16_t, __VA_ARGS__) }                                                 \
    } else {                                                                                                    \
        if (scale_dtype == MTL_F32) { MTL_W4_Z(KERNEL, uint16_t, float, __VA_ARGS__) }                          \
        else { MTL_W4_Z(KERNEL, uint16_t, uint16_t, __VA_ARGS__) }                                              \
    }

// the checks both entry points share (0: passed)
int check_w4(const char* who, const void* codes, const void* scales, int64_t N, int64_t K, int group, int dtype,
             int scale_dtype) {
    const char* bad = nullptr;
    if (N < 1 || K < 1 || N > int64_t(1) << 27 || K > int64_t(1) << 20) bad = "N must be in [1, 2^27], K in [1, 2^20]";
    else if (group != 32 && group != 64 && group != 128) bad = "group must be 32, 64 or 128";
    else if ((dtype != MTL_F32 && dtype != MTL_BF16) || (scale_dtype != MTL_F32 && scale_dtype != MTL_BF16))
        bad = "dtype and scale_dtype must be MTL_F32 or MTL_BF16";
    else if (!codes || !scales) bad = "null pointer";
    else if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) % 16 != 0)
        bad = "codes and scales must be 16-byte aligned";
    if (!bad) return 0;
    set_error(std::string(who) + ": " + bad);
    return MTL_EINVAL;
}

}  // namespace
}  // namespace mtl

extern "C" int mtl_linear_w4(const mtl_linear_w4_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    const int group = p->group, dtype = p->dtype, scale_dtype = p->scale_dtype;
    if (int rc = check_w4(__func__, p->codes, p->scales, p->N, p->K, group, dtype, scale_dtype)) return rc;
    MTL_REQUIRE(p->M >= 0 && p->M <= 64, "M must be in [0, 64]");
    if (p->M == 0) return MTL_OK;
    MTL_REQUIRE(p->x && p->y, "null pointer");
    MTL_REQUIRE(p->ldx >= p->K && p->ldy >= p->N, "rows of x and y must not overlap");
    MTL_REQUIRE(reinterpret_cast<uintptr_t>(p->zeros) % 4 == 0, "zeros must be 4-byte aligned");
    const W4Args a{p->x, p->codes, p->scales, p->zeros, p->bias, p->y, p->ldx, p->ldy, (int)p->M, (int)p->N, (int)p->K,
                   (int)((p->K + kBlockK - 1) / kBlockK)};
    const int tiles = (int)((p->N + kTileRows - 1) / kTileRows);
    MTL_W4(linear_w4_kernel, dim3(tiles), dim3(256), 0, as_stream(stream), a)
    return check_launch("linear_w4");
}

extern "C" int mtl_dequantize_w4(const uint8_t* codes, const void* scales, const uint8_t* zeros, void* W, int64_t ldw,
                                 int64_t N, int64_t K, int32_t group, int32_t dtype, int32_t scale_dtype,
                                 mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    if (int rc = check_w4(__func__, codes, scales, N, K, group, dtype, scale_dtype)) return rc;
    MTL_REQUIRE(W, "null pointer");
    MTL_REQUIRE(ldw >= K, "rows of W must not overlap");
    MTL_REQUIRE(reinterpret_cast<uintptr_t>(zeros) % 4 == 0, "zeros must be 4-byte aligned");
    const W4Args a{nullptr, codes, scales, zeros, nullptr, W, 0, ldw, 0, (int)N, (int)K,
                   (int)((K + kBlockK - 1) / kBlockK)};
    const int64_t tiles = (N + kTileRows - 1) / kTileRows;
    const dim3 grid((a.KB + 3) / 4, (unsigned)std::min<int64_t>(tiles, 65535), (unsigned)((tiles + 65534) / 65535));
    MTL_W4(dequantize_w4_kernel, grid, dim3(256), 0, as_stream(stream), a)
    return check_launch("dequantize_w4");
}
