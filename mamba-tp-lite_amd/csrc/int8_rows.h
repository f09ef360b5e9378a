// A row of floats in codes, on the device, shared by int8.hip and int8_row_linear.hip.
#pragma once

#include "int8.h"

namespace mtl {

// 127 t / a to the nearest whole number: 127 t is exact in 64 bits, and the quotient's rounding there crosses no border
// (one that is no half is 2^-33 or more from it).
__device__ __forceinline__ int code_of(float t, float a) { return (int)rint((double)t * 127.0 / (double)a); }

// The same without 64 bits, for a in [kLeast, kMost] and inv = 127 / a rounded: t inv is off by less than 2e-5, so its
// rounding is the code unless it comes within 3e-5 of a half h = c + 1/2.  There the sign of 127 |t| - h a decides, and is
// exact: 127 |t| = p + pl in two floats; p and h a are whole multiples of a quarter of an ulp of a and 2^12 of those apart at
// most, so their difference is a float, and a rounded sum of two floats has the sign of the sum.
constexpr float kLeast = 0x1p-90f, kMost = 0x1p120f, kNear = 0.5f - 3e-5f;
__device__ __forceinline__ float near_code(float t, float a, float q) {
#pragma clang fp contract(off)
    const float c = floorf(fabsf(q)), u = fabsf(t), p = 127.f * u, pl = fmaf(127.f, u, -p);
    const float e = fmaf(-(c + 0.5f), a, p) + pl;
    const float up = e > 0.f || (e == 0.f && ((int)c & 1)) ? c + 1.f : c;
    return copysignf(up, t);
}

constexpr int kRun = 8;                    // columns a lane takes at a time
typedef float F4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t U4u __attribute__((ext_vector_type(4), aligned(2)));

// a run's first n values, all 8 in whole 16-byte accesses at any alignment; zeros behind n.  (Value by value where rows do not
// start on 16 bytes, 32768 rows of 777 took three times as long as of 768.)
__device__ __forceinline__ void load_run(const float* p, int n, float* v) {
    if (n >= kRun) {
        const F4u lo = *reinterpret_cast<const F4u*>(p), hi = *reinterpret_cast<const F4u*>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = lo[j]; v[4 + j] = hi[j]; }
    } else {
#pragma unroll
        for (int j = 0; j < kRun; ++j) v[j] = j < n ? p[j] : 0.f;
    }
}
__device__ __forceinline__ void load_run(const uint16_t* p, int n, float* v) {
    if (n >= kRun) {
        const U4u x = *reinterpret_cast<const U4u*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(x[j] << 16); v[2 * j + 1] = __uint_as_float(x[j] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int j = 0; j < kRun; ++j) v[j] = j < n ? bf16_to_f32(p[j]) : 0.f;
    }
}

// a row's scale from its largest magnitude's bits (NaN for a row that holds an infinity or NaN) and the norm's factor
__device__ __forceinline__ float row_scale(uint32_t most, float r) {
    return most < 0x7f800000u ? __uint_as_float(most) * r / 127.f : __uint_as_float(0x7fc00000u);
}

// 8 codes of a row of largest magnitude a, as 8 bytes (exact: a is outside [kLeast, kMost]).  One fma rounds t inv + 1.5 2^23
// to a whole number whose low byte is the code.  (t inv rounded, its nearest whole number and that as an integer, with one
// maximum of magnitudes in place of two of bits: 32768 x 2048 in bf16 41 us; 35 now.)
__device__ __forceinline__ uint2 run_codes(const float* t, float a, float inv, bool exact) {
#pragma clang fp contract(off)
    constexpr float kWhole = 12582912.f;
    float c[kRun];
    if (exact) {
#pragma unroll 1
        for (int j = 0; j < kRun; ++j) c[j] = (float)code_of(t[j], a) + kWhole;
    } else {
        float off = 0.f;
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
            c[j] = fmaf(t[j], inv, kWhole);
            off = fmaxf(off, fabsf(fmaf(t[j], inv, kWhole - c[j])));
        }
        if (off > kNear) {
#pragma unroll
            for (int j = 0; j < kRun; ++j)
                if (fabsf(fmaf(t[j], inv, kWhole - c[j])) > kNear) c[j] = near_code(t[j], a, t[j] * inv) + kWhole;
        }
    }
    uint32_t b[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(c[4 * h + 1]), __float_as_uint(c[4 * h]), 0x0c0c0400);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(c[4 * h + 3]), __float_as_uint(c[4 * h + 2]), 0x04000c0c);
        b[h] = lo | hi;
    }
    return uint2{b[0], b[1]};
}

}  // namespace mtl
