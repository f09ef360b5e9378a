// Rows in 8-bit integers (gfx950): floats into codes with a scale for each row, the residual add and RMSNorm with such
// an output, products of two such matrices, and the floats that they stand for.
//   a = max_k |t[k]|,  code[k] = the whole number nearest to 127 t[k] / a (halves to the even one),  scale = a / 127
//   y[m, n] = bias[n] + sx[m] sw[n] sum_k cx[m, k] cw[n, k]
//
// Layout: a row of K codes takes K rounded up to 128 bytes, zeros past K, so no product needs to know where K ends.
// Sums of products are exact in 32 bits: 2^14 K < 2^31 for K < 2^17.

#include "common.h"

namespace mtl {
namespace {

constexpr int kPad = 128;                  // bytes that rows are rounded up to
constexpr int64_t kMaxK = (1 << 17) - 1;

__host__ __device__ inline int64_t padded(int64_t k) { return (k + kPad - 1) / kPad * kPad; }

typedef int I4 __attribute__((ext_vector_type(4)));

// 127 t / a to the nearest whole number: 127 t is exact in 64 bits, and the quotient's rounding there crosses no border
// (one that is no half is 2^-33 or more from it)
__device__ __forceinline__ int code_of(float t, float a) { return (int)rint((double)t * 127.0 / (double)a); }

struct RowsArgs {
    const void* x;             // [M, ldx]
    int64_t ldx;
    const void* y;             // [M, K] to add to x, or null
    float* x_out;              // [M, K], x + y, or null
    const void* w;             // [K]
    int8_t* codes;             // [M, padded(K)]
    float* scales;             // [M]
    int K, Kp;
    float eps;
};

constexpr int kThreads = 256;

template <typename V, typename F> __device__ __forceinline__ V block_reduce(V v, V* s, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) s[wave] = v;
    __syncthreads();
    V r = s[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) r = f(r, s[i]);
    return r;
}

// One workgroup per row.
template <typename T, typename Y, typename W, bool NORM>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const RowsArgs p) {
#pragma clang fp contract(off)
    __shared__ uint32_t s_max[kThreads / 64];
    __shared__ float s_sum[kThreads / 64];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const Y* y = p.y ? static_cast<const Y*>(p.y) + row * p.K : nullptr;
    auto stored = [&](int k) { return y ? Act<T>::load(x + k) + Act<Y>::load(y + k) : Act<T>::load(x + k); };
    auto weighted = [&](float h, int k) { return NORM ? h * Act<W>::load(static_cast<const W*>(p.w) + k) : h; };
    uint32_t most = 0;
    float ss = 0.f;
    for (int k = threadIdx.x; k < p.K; k += kThreads) {
        const float h = stored(k);
        ss = fmaf(h, h, ss);
        most = max(most, abs_bits(weighted(h, k)));
    }
    most = block_reduce(group_umax<64>(most), s_max, [](uint32_t u, uint32_t v) { return max(u, v); });
    float r = 1.f;
    if constexpr (NORM)
        r = rsqrtf(block_reduce(group_sum<64>(ss), s_sum, [](float u, float v) { return u + v; }) / (float)p.K + p.eps);
    const bool finite = most < 0x7f800000u;
    const float a = __uint_as_float(most);
    if (threadIdx.x == 0) p.scales[row] = finite ? a * r / 127.f : __uint_as_float(0x7fc00000u);
    int8_t* codes = p.codes + row * p.Kp;
    for (int k = threadIdx.x; k < p.Kp; k += kThreads) {
        int c = 0;
        if (k < p.K) {
            const float h = stored(k);
            if (p.x_out) p.x_out[row * p.K + k] = h;
            if (finite && most) c = code_of(weighted(h, k), a);
        }
        codes[k] = (int8_t)c;
    }
}

template <typename T> __global__ void __launch_bounds__(kThreads)
dequantize_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ out, int64_t ld,
                  int K, int Kp) {
    const int64_t row = blockIdx.x;
    const float s = scales[row];
    for (int k = threadIdx.x; k < K; k += kThreads) Act<T>::store(out + row * ld + k, (float)codes[row * Kp + k] * s);
}

struct LinearArgs {
    const int8_t* x; const float* sx;      // [M, Kp], [M]
    const int8_t* w; const float* sw;      // [N, Kp], [N]
    const void* bias;                      // [N] or null
    void* y;
    int64_t ldy;
    int M, N, Kp;
};

template <typename T> __device__ __forceinline__ float scaled(int acc, float sx, float sw, float bias) {
    return fmaf((float)acc * sx, sw, bias);
}

// A wavefront takes 16 x 16 outputs: rows of W as the first operand, so a lane holds 4 neighbouring columns of y.
template <typename T> __global__ void __launch_bounds__(kThreads) linear_tile_kernel(const LinearArgs p) {
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int tn = (p.N + 63) / 64;
    const int64_t n0 = ((int64_t)(blockIdx.x % tn) * 4 + (threadIdx.x >> 6)) * 16;
    const int m0 = blockIdx.x / tn * 16;
    if (n0 >= p.N) return;
    const int8_t* x = p.x + (int64_t)min(m0 + r, p.M - 1) * p.Kp + j * 16;
    const int8_t* w = p.w + min(n0 + r, (int64_t)p.N - 1) * p.Kp + j * 16;
    I4 acc = {0, 0, 0, 0};
    for (int k = 0; k < p.Kp; k += 64)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const I4*>(w + k), *reinterpret_cast<const I4*>(x + k),
                                                    acc, 0, 0, 0);
    const int m = m0 + r;
    if (m >= p.M) return;
    const float sx = p.sx[m];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t n = n0 + 4 * j + q;
        if (n >= p.N) return;
        const float b = p.bias ? Act<T>::load(static_cast<const T*>(p.bias) + n) : 0.f;
        Act<T>::store(static_cast<T*>(p.y) + m * p.ldy + n, scaled<T>(acc[q], sx, p.sw[n], b));
    }
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool act(int32_t dtype) { return dtype == MTL_F32 || dtype == MTL_BF16; }

#define MTL_SIZES(M, K)                                                                                    \
    MTL_REQUIRE((M) >= 0 && (M) < (int64_t(1) << 31), "rows must be in [0, 2^31)");                        \
    MTL_REQUIRE((K) >= 1 && (K) <= kMaxK, "K must be in [1, 2^17 - 1]")

}  // namespace
}  // namespace mtl

extern "C" int mtl_quantize_int8(const void* x, int64_t ldx, int8_t* codes, float* scales, int64_t M, int64_t K,
                                 int32_t dtype, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_SIZES(M, K);
    MTL_REQUIRE(act(dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (M == 0) return MTL_OK;
    MTL_REQUIRE(x && codes && scales, "null pointer");
    MTL_REQUIRE(ldx >= 0, "ldx must not be negative");
    MTL_REQUIRE(al16(codes), "codes must be 16-byte aligned");
    RowsArgs a{};
    a.x = x; a.ldx = ldx; a.codes = codes; a.scales = scales; a.K = (int)K; a.Kp = (int)padded(K);
    const dim3 grid((unsigned)M), nt(kThreads);
    if (dtype == MTL_F32) hipLaunchKernelGGL((quantize_kernel<float, float, float, false>), grid, nt, 0, as_stream(stream), a);
    else hipLaunchKernelGGL((quantize_kernel<uint16_t, float, float, false>), grid, nt, 0, as_stream(stream), a);
    return check_launch("quantize_int8");
}

extern "C" int mtl_add_rmsnorm_int8(const mtl_add_rmsnorm_int8_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    MTL_SIZES(p->M, p->K);
    MTL_REQUIRE(act(p->y_dtype) && act(p->w_dtype), "y_dtype and w_dtype must be MTL_F32 or MTL_BF16");
    if (p->M == 0) return MTL_OK;
    MTL_REQUIRE(p->x && p->w && p->codes && p->scales, "null pointer");
    MTL_REQUIRE(al16(p->codes), "codes must be 16-byte aligned");
    RowsArgs a{};
    a.x = p->x; a.ldx = p->K; a.y = p->y; a.x_out = p->x_out; a.w = p->w; a.codes = p->codes; a.scales = p->scales;
    a.K = (int)p->K; a.Kp = (int)padded(p->K); a.eps = p->eps;
    const dim3 grid((unsigned)p->M), nt(kThreads);
    const bool yb = p->y_dtype == MTL_BF16, wb = p->w_dtype == MTL_BF16;
#define MTL_NORM8(Y, W) hipLaunchKernelGGL((quantize_kernel<float, Y, W, true>), grid, nt, 0, as_stream(stream), a)
    if (yb) { if (wb) MTL_NORM8(uint16_t, uint16_t); else MTL_NORM8(uint16_t, float); }
    else { if (wb) MTL_NORM8(float, uint16_t); else MTL_NORM8(float, float); }
#undef MTL_NORM8
    return check_launch("add_rmsnorm_int8");
}

extern "C" int mtl_dequantize_int8(const int8_t* codes, const float* scales, void* out, int64_t ldo, int64_t M, int64_t K,
                                   int32_t dtype, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_SIZES(M, K);
    MTL_REQUIRE(act(dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (M == 0) return MTL_OK;
    MTL_REQUIRE(codes && scales && out, "null pointer");
    MTL_REQUIRE(al16(codes), "codes must be 16-byte aligned");
    MTL_REQUIRE(ldo >= K, "rows of out must not overlap");
    const dim3 grid((unsigned)M), nt(kThreads);
    if (dtype == MTL_F32)
        hipLaunchKernelGGL((dequantize_kernel<float>), grid, nt, 0, as_stream(stream), codes, scales, static_cast<float*>(out),
                           ldo, (int)K, (int)padded(K));
    else
        hipLaunchKernelGGL((dequantize_kernel<uint16_t>), grid, nt, 0, as_stream(stream), codes, scales,
                           static_cast<uint16_t*>(out), ldo, (int)K, (int)padded(K));
    return check_launch("dequantize_int8");
}

extern "C" int mtl_linear_int8(const mtl_linear_int8_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    MTL_SIZES(p->M, p->K);
    MTL_REQUIRE(p->N >= 1 && p->N <= int64_t(1) << 27, "N must be in [1, 2^27]");
    MTL_REQUIRE(act(p->dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (p->M == 0) return MTL_OK;
    MTL_REQUIRE(p->x && p->x_scales && p->w && p->w_scales && p->y, "null pointer");
    MTL_REQUIRE(al16(p->x) && al16(p->w), "codes must be 16-byte aligned");
    MTL_REQUIRE(p->ldy >= p->N, "rows of y must not overlap");
    const int64_t tiles = ((p->N + 63) / 64) * ((p->M + 15) / 16);
    MTL_REQUIRE(tiles < (int64_t(1) << 31), "too many output tiles");
    const LinearArgs a{p->x, p->x_scales, p->w, p->w_scales, p->bias, p->y, p->ldy, (int)p->M, (int)p->N, (int)padded(p->K)};
    const dim3 grid((unsigned)tiles), nt(kThreads);
    if (p->dtype == MTL_F32) hipLaunchKernelGGL((linear_tile_kernel<float>), grid, nt, 0, as_stream(stream), a);
    else hipLaunchKernelGGL((linear_tile_kernel<uint16_t>), grid, nt, 0, as_stream(stream), a);
    return check_launch("linear_int8");
}
