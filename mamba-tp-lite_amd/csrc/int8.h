// The layout of rows in 8-bit integers, shared by int8.hip and int8_linear.hip.
//
// A row of K codes takes K rounded up to 128 bytes, zeros past K, so no product needs to know where K ends.  Sums of
// products of codes are exact in 32 bits: 2^14 K < 2^31 for K < 2^17.
#pragma once

#include <algorithm>

#include "common.h"

namespace mtl {

constexpr int kInt8Pad = 128;              // bytes that rows are rounded up to
constexpr int64_t kInt8MaxK = (1 << 17) - 1;

inline int64_t int8_row(int64_t k) { return (k + kInt8Pad - 1) / kInt8Pad * kInt8Pad; }
inline bool act_dtype(int32_t dtype) { return dtype == MTL_F32 || dtype == MTL_BF16; }

// Where mtl_row_linear_int8 takes a row and is no slower than two launches.  Its workgroups of 16 columns of y each put the
// row into codes again, which pays while there are few or their rows of W long; two launches read a wide W at 5.5 TB/s, but at
// 4.3-4.9 where its rows are a power of two apart, and one at 5.1.  us of one / of two, fp32, W from HBM, out of 160 sizes:
// 8192x64 4.4 / 4.5, 9216x64 5.6 / 4.6; 12288x512 6.1 / 6.6, 20480x512 8.0 / 7.3; 16384x768 7.1 / 7.0, 24576x768 9.1 / 8.8;
// 24576x1024 9.1 / 9.6, 32768x1024 11.3 / 10.7; 50280x2048 19.4 / 21.6, 65536x4096 48.7 / 55.0; 16384x2560 11.5 / 13.6, 24576x2560
// 16.0 / 15.7; 16384x7168 25.4 / 26.9, 20480x7168 33.2 / 30.0.  With a norm: 8192x256 5.2 / 5.3, 12288x256 6.8 / 6.2; 12288x768 6.9 /
// 7.0, 16384x768 8.1 / 7.5; 16384x4096 16.5 / 18.1, 24576x2560 18.4 / 16.4.
inline bool row_linear_int8_pays(int64_t n, int64_t k, bool norm) {
    if (k < 1 || k > (norm ? 4096 : 8192)) return false;
    const int64_t kp = int8_row(k), wide = norm || (kp & (kp - 1)) ? 16384 : 65536;
    return n >= 1 && n <= std::min(std::max<int64_t>(8192, (norm ? 16 : 25) * k), wide);
}

// whether two runs of bytes meet (a null one is empty)
inline bool meet(const void* a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p && q && p < q + (uintptr_t)nb && q < p + (uintptr_t)na;
}

// f(first row, rows, blocks) for each of the launches that M rows take, `per` of them to a block of `threads`: a launch has
// fewer than 2^32 threads.
template <typename F> int in_launches(int64_t M, int64_t per, int threads, F&& f) {
    const int64_t most = ((int64_t(1) << 32) - 1) / threads * per;
    for (int64_t m = 0; m < M; m += most) {
        const int64_t rows = std::min(most, M - m);
        if (const int rc = f(m, rows, (unsigned)((rows + per - 1) / per))) return rc;
    }
    return MTL_OK;
}

#define MTL_INT8_SIZES(M, K)                                                        \
    MTL_REQUIRE((M) >= 0 && (M) < (int64_t(1) << 31), "rows must be in [0, 2^31)"); \
    MTL_REQUIRE((K) >= 1 && (K) <= kInt8MaxK, "K must be in [1, 2^17 - 1]")

typedef int I4 __attribute__((ext_vector_type(4)));

// the float of a sum, each factor rounded once
__device__ __forceinline__ float scaled(int acc, float sx, float sw, float bias) { return fmaf((float)acc * sx, sw, bias); }

}  // namespace mtl
