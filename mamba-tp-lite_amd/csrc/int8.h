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

// Where mtl_row_linear_int8 takes a row and is no slower than two launches (us, fp32: N x K of 16384x768 7.3 for 7.9,
// 24000x768 9.3 for 8.1, 50280x768 16.4 for 12.0; 24000x2048 11.1 for 13.4).
inline bool row_linear_int8_pays(int64_t n, int64_t k, bool norm) { return k <= (norm ? 4096 : 8192) && n <= 16384; }

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
