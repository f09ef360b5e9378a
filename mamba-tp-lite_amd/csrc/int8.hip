// Rows in 8-bit integers (gfx950): floats into codes with a scale for each row, the residual add and RMSNorm with such
// an output, and the floats that they stand for.  int8_linear.hip multiplies them.
//   a = max_k |t[k]|,  code[k] = the whole number nearest to 127 t[k] / a (halves to the even one),  scale = a / 127

#include "int8_rows.h"

namespace mtl {
namespace {

struct RowsArgs {
    const void* x;             // [M, ldx]
    int64_t ldx;
    const void* y;             // [M, K] to add to x, or null
    float* x_out;              // [M, K], x + y, or null
    const void* w;             // [K]
    int8_t* codes;             // [M, Kp]
    float* scales;             // [M]
    int64_t M;
    int K, Kp;
    float eps;
};

// Rows held in registers from one pass over memory: as many wavefronts to a row as RU runs of 8 columns a lane need, or ONE.
// HBM is the bound.
constexpr int kRowThreads = 512;
template <typename T, typename Y, typename W, bool NORM, bool ONE, int RU>
__global__ void __launch_bounds__(ONE ? 256 : kRowThreads) quantize_kernel(const RowsArgs p) {
#pragma clang fp contract(off)
    constexpr int NW = ONE ? 4 : kRowThreads / 64;
    const int G = ONE ? 64 : (int)blockDim.x;
    __shared__ uint32_t s_max[NW];
    __shared__ float s_sum[NW];
    __shared__ __align__(16) float s_out[NORM ? NW : 1][64 * kRun];
    const int64_t row = ONE ? (int64_t)blockIdx.x * 4 + threadIdx.x / 64 : blockIdx.x;
    const int t = ONE ? threadIdx.x % 64 : threadIdx.x;
    if (row >= p.M) return;                                   // (whole wavefronts)
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const bool add = NORM && p.y;
    float v[RU][kRun], wv[RU][kRun];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int k = (u * G + t) * kRun, kc = min(k, (p.K - 1) / kRun * kRun);
        load_run(x + kc, p.K - kc, v[u]);
        if constexpr (NORM) load_run(static_cast<const W*>(p.w) + kc, p.K - kc, wv[u]);
    }
    if (add) {
        const Y* y = static_cast<const Y*>(p.y) + row * p.K;
        float yv[RU][kRun];
#pragma unroll
        for (int u = 0; u < RU; ++u) {
            const int k = (u * G + t) * kRun, kc = min(k, (p.K - 1) / kRun * kRun);
            load_run(y + kc, p.K - kc, yv[u]);
        }
#pragma unroll
        for (int u = 0; u < RU; ++u)
#pragma unroll
            for (int j = 0; j < kRun; ++j) v[u][j] += yv[u][j];
    }
    if constexpr (NORM) {
        if (p.x_out) {
            // through LDS, so that an instruction stores whole lines: 32768 x 2048 with bf16 y 135 -> 121 us (6.1 TB/s).  Past the
            // caches, as it is read again a layer later only: into another buffer 131 without; in place 129, 128 with it, and with
            // the product behind it level from 32 rows to 32768.
            const int lane = t & 63, k0 = (t - lane) * kRun;
            float* s = s_out[threadIdx.x / 64];
#pragma unroll
            for (int u = 0; u < RU; ++u) {
                st4(s + lane * kRun, F4v{v[u][0], v[u][1], v[u][2], v[u][3]});
                st4(s + lane * kRun + 4, F4v{v[u][4], v[u][5], v[u][6], v[u][7]});
                wave_lds_fence();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int at = 256 * i + 4 * lane, k = u * G * kRun + k0 + at;
                    const F4v o = ld4(s + at);
                    float* d = p.x_out + row * p.K + k;
                    if (k + 4 <= p.K) {
                        __builtin_nontemporal_store(F4u{o[0], o[1], o[2], o[3]}, reinterpret_cast<F4u*>(d));
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (k + j < p.K) d[j] = o[j];
                    }
                }
                wave_lds_fence();
            }
        }
    }
    int above = 0;                                            // bits of the largest positive value and of the least
    uint32_t below = 0;                                       // negative one (of the largest, where there is none)
    float ss = 0.f;
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int k = (u * G + t) * kRun;
        if (k < p.K) {
#pragma unroll
            for (int j = 0; j < kRun; ++j) {
                if constexpr (NORM) {
                    ss = fmaf(v[u][j], v[u][j], ss);
                    v[u][j] *= wv[u][j];
                }
                const uint32_t b = __float_as_uint(v[u][j]);
                above = max(above, (int)b);
                below = max(below, b);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kRun; ++j) v[u][j] = 0.f;
        }
    }
    uint32_t most = group_umax<64>(max((uint32_t)above, below & 0x7fffffffu));
    if constexpr (NORM) ss = group_sum<64>(ss);
    if constexpr (!ONE) {
        if (t % 64 == 0) {
            s_max[t / 64] = most;
            s_sum[t / 64] = ss;
        }
        lds_barrier();
        most = s_max[0];
        ss = s_sum[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) {
            if (i >= G / 64) break;
            most = max(most, s_max[i]);
            ss += s_sum[i];
        }
    }
    const float r = NORM ? rsqrtf(ss / (float)p.K + p.eps) : 1.f;
    if (t == 0) p.scales[row] = row_scale(most, r);
    const bool none = most == 0 || most >= 0x7f800000u;
    const float a = __uint_as_float(most), inv = 127.f / a;
    const bool exact = a < kLeast || a > kMost;
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int k = (u * G + t) * kRun;
        if (k < p.Kp) {
            const uint2 c = none ? uint2{0, 0} : run_codes(v[u], a, inv, exact);
            // (kept in the caches for the product that reads them next.  Past them a call alone over the same floats is up to a
            // sixth faster, fp32 32768 x 2048 56 -> 47 us, but slower from HBM, 32768 x 1536 43.3 -> 45.5, and with its reader, 16384
            // x 1536 through [768, 1536] 46.4 -> 48.7, 1024 rows 10.8 -> 11.5, with the values 42.0 -> 45.1)
            *reinterpret_cast<uint2*>(p.codes + row * p.Kp + k) = c;
        }
    }
}

// Longer rows: one workgroup each, read twice.
constexpr int kLongThreads = 1024;
template <typename T, typename Y, typename W, bool NORM>
__global__ void __launch_bounds__(kLongThreads) quantize_long_kernel(const RowsArgs p) {
#pragma clang fp contract(off)
    constexpr int NW = kLongThreads / 64;
    __shared__ uint32_t s_max[NW];
    __shared__ float s_sum[NW];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const Y* y = NORM && p.y ? static_cast<const Y*>(p.y) + row * p.K : nullptr;
    auto load = [&](int k, float* v) {
        load_run(x + k, p.K - k, v);
        if (y) {
            float yv[kRun];
            load_run(y + k, p.K - k, yv);
#pragma unroll
            for (int j = 0; j < kRun; ++j) v[j] += yv[j];
        }
    };
    auto weigh = [&](int k, float* v) {
        if constexpr (NORM) {
            float wv[kRun];
            load_run(static_cast<const W*>(p.w) + k, p.K - k, wv);
#pragma unroll
            for (int j = 0; j < kRun; ++j) v[j] *= wv[j];
        }
    };
    uint32_t most = 0;
    float ss = 0.f, v[kRun];
    for (int k = threadIdx.x * kRun; k < p.K; k += kLongThreads * kRun) {
        load(k, v);
#pragma unroll
        for (int j = 0; j < kRun; ++j) ss = fmaf(v[j], v[j], ss);
        weigh(k, v);
#pragma unroll
        for (int j = 0; j < kRun; ++j) most = max(most, abs_bits(v[j]));
    }
    most = group_umax<64>(most);
    ss = group_sum<64>(ss);
    if (threadIdx.x % 64 == 0) {
        s_max[threadIdx.x / 64] = most;
        s_sum[threadIdx.x / 64] = ss;
    }
    lds_barrier();
    most = s_max[0];
    ss = s_sum[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
        most = max(most, s_max[i]);
        ss += s_sum[i];
    }
    const float r = NORM ? rsqrtf(ss / (float)p.K + p.eps) : 1.f;
    if (threadIdx.x == 0) p.scales[row] = row_scale(most, r);
    const bool none = most == 0 || most >= 0x7f800000u;
    const float a = __uint_as_float(most), inv = 127.f / a;
    const bool exact = a < kLeast || a > kMost;
    for (int k = threadIdx.x * kRun; k < p.Kp; k += kLongThreads * kRun) {
        uint2 c{0, 0};
        if (k < p.K) {
            load(k, v);
            if (NORM && p.x_out) {                            // (x and y, which it may be, are read before)
#pragma unroll
                for (int j = 0; j < kRun; ++j)
                    if (k + j < p.K) p.x_out[row * p.K + k + j] = v[j];
            }
            weigh(k, v);
            if (!none) c = run_codes(v, a, inv, exact);
        }
        *reinterpret_cast<uint2*>(p.codes + row * p.Kp + k) = c;
    }
}

template <typename T, typename Y, typename W, bool NORM> int launch_rows(const RowsArgs& a, hipStream_t st) {
    auto go = [&](void (*kernel)(RowsArgs), int per, int threads) {
        return in_launches(a.M, per, threads, [&](int64_t m, int64_t rows, unsigned blocks) {
            RowsArgs c = a;
            c.x = static_cast<const T*>(a.x) + m * a.ldx;
            if (a.y) c.y = static_cast<const Y*>(a.y) + m * a.K;
            if (a.x_out) c.x_out = a.x_out + m * a.K;
            c.codes = a.codes + m * a.Kp;
            c.scales = a.scales + m;
            c.M = rows;
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3((unsigned)threads), 0, st, c);
            return check_launch(NORM ? "add_rmsnorm_int8" : "quantize_int8");
        });
    };
#define MTL_ROWS(ONE, RU) \
    go(quantize_kernel<T, Y, W, NORM, ONE, RU>, ONE ? 4 : 1, ONE ? 256 : (a.Kp + 512 * RU - 1) / (512 * RU) * 64)
    // A wavefront to a row of up to 1024 columns where there are many; otherwise so many that a lane has one run, or two or
    // four of long rows.  us: norms of 32768 x 2048 with bf16 y 148 with a wavefront, 133 with four; 32768 x 768 58, 60; rows
    // of 4096 in bf16, 32768 of them 71 with two runs, 83 with one; 8 of them 3.5, 3.1; 8192 x 8192 34 with two, 36 with four.
    if (a.Kp <= 512 && a.M >= 1024) return MTL_ROWS(true, 1);
    if (a.Kp <= 1024 && a.M >= 1024) return MTL_ROWS(true, 2);
    if (a.Kp <= (a.M <= 1024 ? 4096 : 2048)) return MTL_ROWS(false, 1);
    if (a.Kp <= 8192) return MTL_ROWS(false, 2);
    if (a.Kp <= 16384) return MTL_ROWS(false, 4);
    return go(quantize_long_kernel<T, Y, W, NORM>, 1, kLongThreads);
#undef MTL_ROWS
}

typedef uint32_t U4v __attribute__((ext_vector_type(4)));

// A wavefront reads runs of R codes of a row and writes 16 bytes a lane; PAST: past the L2s.
template <typename T, bool VEC, bool PAST = false> __global__ void __launch_bounds__(256)
dequantize_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ out, int64_t ld,
                  int64_t M, int K, int Kp) {
    constexpr int R = VEC ? 16 / (int)sizeof(T) : 1, U = VEC ? 4 : 8;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    const int k0 = (int)blockIdx.y * (64 * R * U) + (threadIdx.x & 63) * R;
    const float s = scales[row];
    const int8_t* c = codes + row * Kp;
    T* o = out + row * ld;
    if constexpr (VEC) {
        uint2 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(k0 + u * 64 * R, Kp - R);
            if constexpr (R == 4) q[u].x = *reinterpret_cast<const uint32_t*>(c + k);
            else q[u] = *reinterpret_cast<const uint2*>(c + k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * 64 * R;
            float f[8];
#pragma unroll
            for (int j = 0; j < R; ++j) f[j] = (float)(int8_t)((j < 4 ? q[u].x : q[u].y) >> (8 * (j & 3))) * s;
            if (k + R <= K) {
                U4v v;
                if constexpr (R == 4) v = U4v{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
                else v = U4v{f32x2_to_bf16x2(f[0], f[1]), f32x2_to_bf16x2(f[2], f[3]), f32x2_to_bf16x2(f[4], f[5]),
                             f32x2_to_bf16x2(f[6], f[7])};
                if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<U4v*>(o + k));
                else *reinterpret_cast<U4v*>(o + k) = v;
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (k + j < K) Act<T>::store(o + k + j, f[j]);
            }
        }
    } else {
        int8_t q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = c[min(k0 + u * 64, Kp - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u * 64 < K) Act<T>::store(o + k0 + u * 64, (float)q[u] * s);
    }
}

}  // namespace
}  // namespace mtl

extern "C" int mtl_quantize_int8(const void* x, int64_t ldx, int8_t* codes, float* scales, int64_t M, int64_t K,
                                 int32_t dtype, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_INT8_SIZES(M, K);
    MTL_REQUIRE(act_dtype(dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (M == 0) return MTL_OK;
    MTL_REQUIRE(x && codes && scales, "null pointer");
    MTL_REQUIRE(ldx >= 0, "ldx must not be negative");
    MTL_REQUIRE(al16(codes), "codes must be 16-byte aligned");
    RowsArgs a{};
    a.x = x; a.ldx = ldx; a.codes = codes; a.scales = scales; a.M = M; a.K = (int)K; a.Kp = (int)int8_row(K);
    return dtype == MTL_F32 ? launch_rows<float, float, float, false>(a, as_stream(stream))
                            : launch_rows<uint16_t, float, float, false>(a, as_stream(stream));
}

extern "C" int mtl_add_rmsnorm_int8(const mtl_add_rmsnorm_int8_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    MTL_INT8_SIZES(p->M, p->K);
    MTL_REQUIRE(act_dtype(p->y_dtype) && act_dtype(p->w_dtype), "y_dtype and w_dtype must be MTL_F32 or MTL_BF16");
    if (p->M == 0) return MTL_OK;
    MTL_REQUIRE(p->x && p->w && p->codes && p->scales, "null pointer");
    MTL_REQUIRE(al16(p->codes), "codes must be 16-byte aligned");
    if (p->x_out) {
        // (a value's own place is read before it is written; another's may not be)
        const int64_t bytes = 4 * p->M * p->K;
        const bool bf16 = p->y_dtype == MTL_BF16;
        MTL_REQUIRE((p->x_out == p->x || !meet(p->x_out, bytes, p->x, bytes)) &&
                    ((!bf16 && p->x_out == p->y) || !meet(p->x_out, bytes, p->y, bf16 ? bytes / 2 : bytes)) &&
                    !meet(p->x_out, bytes, p->w, (p->w_dtype == MTL_BF16 ? 2 : 4) * p->K),
                    "x_out must be x, a float y, or overlap no operand");
    }
    RowsArgs a{};
    a.x = p->x; a.ldx = p->K; a.y = p->y; a.x_out = p->x_out; a.w = p->w; a.codes = p->codes; a.scales = p->scales;
    a.M = p->M; a.K = (int)p->K; a.Kp = (int)int8_row(p->K); a.eps = p->eps;
    const hipStream_t st = as_stream(stream);
    if (p->y_dtype == MTL_BF16)
        return p->w_dtype == MTL_BF16 ? launch_rows<float, uint16_t, uint16_t, true>(a, st)
                                      : launch_rows<float, uint16_t, float, true>(a, st);
    return p->w_dtype == MTL_BF16 ? launch_rows<float, float, uint16_t, true>(a, st)
                                  : launch_rows<float, float, float, true>(a, st);
}

extern "C" int mtl_dequantize_int8(const int8_t* codes, const float* scales, void* out, int64_t ldo, int64_t M, int64_t K,
                                   int32_t dtype, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_INT8_SIZES(M, K);
    MTL_REQUIRE(act_dtype(dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (M == 0) return MTL_OK;
    MTL_REQUIRE(codes && scales && out, "null pointer");
    MTL_REQUIRE(al16(codes), "codes must be 16-byte aligned");
    MTL_REQUIRE(ldo >= K, "rows of out must not overlap");
    const bool f32 = dtype == MTL_F32, vec = al16(out) && ldo * (f32 ? 4 : 2) % 16 == 0;
    const int per = vec ? f32 ? 1024 : 2048 : 512;            // columns of a workgroup
    const unsigned parts = (unsigned)((K + per - 1) / per);
    auto go = [&](auto* kernel, auto* to) {
        return in_launches(M, 4, 256, [&](int64_t m, int64_t rows, unsigned blocks) {
            hipLaunchKernelGGL(kernel, dim3(blocks, parts), dim3(256), 0, as_stream(stream), codes + m * int8_row(K),
                               scales + m, to + m * ldo, ldo, rows, (int)K, (int)int8_row(K));
            return check_launch("dequantize_int8");
        });
    };
    // Past the L2s from 4 MB on: what they hold is written back when the kernel ends, and from 16 MB on rows read before and values
    // leave each other more of the MALL.  us, kept and past, inputs from HBM and two outputs in turn, these alone / after a norm of
    // the rows / with a reader behind that: fp32 256x2048 (2 MB) 2.5, 2.5 / 6.6, 6.6 / 10.1, 10.2; 2048x2048 (16 MB) 5.6, 4.6 / 17.6,
    // 16.5 / 23.1, 22.3; 4096x2048 8.2, 8.1 / 28.3, 28.2 / 36.8, 37.7; 8192x2048 16.2, 17.4 / 55.7, 51.4 / 67.5, 67.3; 24576x2048 (192 MB)
    // 45.7, 46.5 / 168, 151 / 202, 194.  Over one output again and again, with nothing between, kept ones are up to 15% faster from
    // 48 to 224 MB.
    const bool past = M * ldo * (f32 ? 4 : 2) >= 4 << 20;
    if (f32)
        return go(vec ? past ? dequantize_kernel<float, true, true> : dequantize_kernel<float, true>
                      : dequantize_kernel<float, false>, static_cast<float*>(out));
    return go(vec ? past ? dequantize_kernel<uint16_t, true, true> : dequantize_kernel<uint16_t, true>
                  : dequantize_kernel<uint16_t, false>, static_cast<uint16_t*>(out));
}
