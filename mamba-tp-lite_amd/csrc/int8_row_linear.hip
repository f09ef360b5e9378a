// One float row through a matrix of 8-bit integers in one launch (gfx950): every workgroup puts the row into codes by itself,
// as mtl_quantize_int8 or mtl_add_rmsnorm_int8 does and to the bit, while its first rows of W are on their way from memory.
// us, fp32, W from HBM, the two launches and this one: 8192x2048 7.9 -> 5.8 (the product alone 5.6), with the norm 8.5 -> 6.7;
// 2048x4096 8.0 -> 5.7 and 8.3 -> 7.3; 768x1536 5.0 -> 3.2 and 5.8 -> 4.1.  (Up to 4 rows in the same way: 2048x4096 8.1 ->
// 7.2, with the norm 8.8 -> 13.9: not kept.)

#include "int8_rows.h"

namespace mtl {
namespace {

constexpr int kWaves = 8, kThreads = kWaves * 64;

struct RowLinearArgs {
    const void* x;             // [K]
    const float* add;          // [K] to add to x, or null
    float* x_out;              // [K], x + add, or null
    const void* norm_w;        // [K]
    const int8_t* w; const float* sw;      // [N, Kp], [N]
    const void* bias;          // [N] or null
    void* y;                   // [N]
    int N, K, Kp;
    float eps;
    bool vec;                  // y on 16 bytes
    bool bias_bf16;
};

// T: y; X: x; W: the norm's weight.  A lane holds RU runs of 8 columns (one, and the same as quantize_kernel's, where the
// norm's sum of squares has an order); then the wavefronts take 16 columns of y, as stream_int8_kernel's.
template <typename T, typename X, typename W, bool NORM, int RU>
__global__ void __launch_bounds__(kThreads) row_linear_int8_kernel(const RowLinearArgs p) {
#pragma clang fp contract(off)
    constexpr int U = 2;
    __shared__ __align__(16) int8_t s_x[kThreads * kRun * RU];
    __shared__ __align__(16) I4 s_acc[kWaves][64];
    __shared__ uint32_t s_max[kWaves];
    __shared__ float s_sum[kWaves], s_scale;
    const int t = threadIdx.x, lane = t & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);

    float v[RU][kRun], nw[RU][kRun], add[RU][kRun];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int kc = min((u * kThreads + t) * kRun, (p.K - 1) / kRun * kRun), n = p.K - kc;
        load_run(static_cast<const X*>(p.x) + kc, n, v[u]);
        if constexpr (NORM) {
            load_run(static_cast<const W*>(p.norm_w) + kc, n, nw[u]);
            if (p.add) load_run(p.add + kc, n, add[u]);
        }
    }

    const int n0 = blockIdx.x * 16;
    const int8_t* w = p.w + (int64_t)min(n0 + r16, p.N - 1) * p.Kp + 32 * g4;
    const int steps = p.Kp / 128, per = (steps + kWaves - 1) / kWaves, s0 = wave * per, s1 = min(s0 + per, steps);
    I4 fw[U][2];
    auto load = [&](int u, int s) __attribute__((always_inline)) {
        const int k = min(s, steps - 1) * 128;                  // (past the run: loaded, never used)
#pragma unroll
        for (int h = 0; h < 2; ++h) fw[u][h] = *reinterpret_cast<const I4*>(w + k + 16 * h);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(u, s0 + u);

    uint32_t most = 0;
    float ss = 0.f;
#pragma unroll
    for (int u = 0; u < RU; ++u) {
        const int k = (u * kThreads + t) * kRun;
        if (k < p.K) {
            if constexpr (NORM) {
                if (p.add) {
#pragma unroll
                    for (int j = 0; j < kRun; ++j) v[u][j] += add[u][j];
                }
                if (p.x_out && blockIdx.x == 0) {
#pragma unroll
                    for (int j = 0; j < kRun; ++j)
                        if (k + j < p.K) p.x_out[k + j] = v[u][j];
                }
            }
#pragma unroll
            for (int j = 0; j < kRun; ++j) {
                if constexpr (NORM) {
                    ss = fmaf(v[u][j], v[u][j], ss);
                    v[u][j] *= nw[u][j];
                }
                most = max(most, abs_bits(v[u][j]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < kRun; ++j) v[u][j] = 0.f;
        }
    }
    most = group_umax<64>(most);
    if constexpr (NORM) ss = group_sum<64>(ss);
    if (lane == 0) {
        s_max[wave] = most;
        s_sum[wave] = ss;
    }
    lds_barrier();
    most = s_max[0];
    ss = s_sum[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        most = max(most, s_max[i]);
        ss += s_sum[i];
    }
    if (t == 0) s_scale = row_scale(most, NORM ? rsqrtf(ss / (float)p.K + p.eps) : 1.f);
    const bool none = most == 0 || most >= 0x7f800000u;
    const float a = __uint_as_float(most), inv = 127.f / a;
    const bool exact = a < kLeast || a > kMost;
#pragma unroll
    for (int u = 0; u < RU; ++u)
        *reinterpret_cast<uint2*>(s_x + (u * kThreads + t) * kRun) = none ? uint2{0, 0} : run_codes(v[u], a, inv, exact);
    lds_barrier();

    // (all 16 rows of the matrix instruction's second operand are the one row)
    const int8_t* x = s_x + 32 * g4;
    I4 acc = {0, 0, 0, 0};
    for (int s = s0; s < s1; s += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u < s1) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                        fw[u][h], *reinterpret_cast<const I4*>(x + (s + u) * 128 + 16 * h), acc, 0, 0, 0);
            }
            if (s + U < s1) load(u, s + U + u);
        }
    }
    s_acc[wave][lane] = acc;
    lds_barrier();
    const int n = n0 + 4 * g4;
    if (wave || r16) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) acc += s_acc[i][lane];
    T* y = static_cast<T*>(p.y) + n;
    F4v out;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int nc = min(n + q, p.N - 1);
        out[q] = scaled(acc[q], s_scale, p.sw[nc], p.bias ? load_param(p.bias, nc, p.bias_bf16) : 0.f);
    }
    if (p.vec && n + 4 <= p.N) {
        st4(y, out);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (n + q < p.N) Act<T>::store(y + q, out[q]);
    }
}

template <typename T, typename X> int launch(const RowLinearArgs& a, hipStream_t st) {
    constexpr int kMost = 1 << 26;                             // columns of y: a launch has fewer than 2^32 threads
    if (a.N > kMost) {
        RowLinearArgs c = a;
        c.N = kMost;
        if (const int rc = launch<T, X>(c, st)) return rc;
        c = a;
        c.x_out = nullptr;
        c.w += (int64_t)kMost * a.Kp;
        c.sw += kMost;
        if (a.bias) c.bias = static_cast<const uint8_t*>(a.bias) + (int64_t)kMost * (a.bias_bf16 ? 2 : 4);
        c.y = static_cast<T*>(a.y) + kMost;
        c.N -= kMost;
        return launch<T, X>(c, st);
    }
    const dim3 grid((unsigned)((a.N + 15) / 16)), nt(kThreads);
    if (a.norm_w) hipLaunchKernelGGL((row_linear_int8_kernel<T, float, X, true, 1>), grid, nt, 0, st, a);
    else if (a.K <= 4096) hipLaunchKernelGGL((row_linear_int8_kernel<T, X, X, false, 1>), grid, nt, 0, st, a);
    else hipLaunchKernelGGL((row_linear_int8_kernel<T, X, X, false, 2>), grid, nt, 0, st, a);
    return check_launch("row_linear_int8");
}

}  // namespace
}  // namespace mtl

extern "C" int mtl_row_linear_int8_pays(int64_t N, int64_t K, int32_t norm) {
    return mtl::row_linear_int8_pays(N, K, norm != 0) ? 1 : 0;
}

extern "C" int mtl_row_linear_int8(const mtl_row_linear_int8_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    MTL_REQUIRE(p->K >= 1 && p->K <= (p->norm_w ? 4096 : 8192), "K must be in [1, 8192], with a norm in [1, 4096]");
    MTL_REQUIRE(p->N >= 1 && p->N <= int64_t(1) << 27, "N must be in [1, 2^27]");
    MTL_REQUIRE(act_dtype(p->dtype), "dtype must be MTL_F32 or MTL_BF16");
    MTL_REQUIRE(p->x && p->w && p->w_scales && p->y, "null pointer");
    MTL_REQUIRE(p->norm_w || !(p->add || p->x_out), "add and x_out need a norm");
    MTL_REQUIRE(al16(p->w), "codes must be 16-byte aligned");
    const bool bf16 = p->dtype == MTL_BF16, f32 = !bf16 || p->y_f32;
    // (every workgroup reads all of the row, while others write)
    const int64_t es = bf16 ? 2 : 4, y_bytes = p->N * (f32 ? 4 : 2), out_bytes = 4 * p->K;
    const struct { const void* at; int64_t bytes; } in[] = {
        {p->x, p->K * (p->norm_w ? 4 : es)}, {p->add, 4 * p->K}, {p->norm_w, es * p->K}, {p->w, p->N * int8_row(p->K)},
        {p->w_scales, 4 * p->N}, {p->bias, es * p->N}};
    for (const auto& i : in) MTL_REQUIRE(!meet(p->x_out, out_bytes, i.at, i.bytes), "x_out must not overlap an operand");
    for (const auto& i : in) MTL_REQUIRE(!meet(p->y, y_bytes, i.at, i.bytes), "y must not overlap an operand");
    MTL_REQUIRE(!meet(p->y, y_bytes, p->x_out, out_bytes), "y must not overlap x_out");
    const RowLinearArgs a{p->x, p->add, p->x_out, p->norm_w, p->w, p->w_scales, p->bias, p->y, (int)p->N, (int)p->K,
                          (int)int8_row(p->K), p->eps, al16(p->y), bf16};
    const hipStream_t st = as_stream(stream);
    return !bf16 ? launch<float, float>(a, st) : f32 ? launch<float, uint16_t>(a, st) : launch<uint16_t, uint16_t>(a, st);
}
