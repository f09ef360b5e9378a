// Log probabilities of given tokens, entropy and the most probable tokens of rows of logits (gfx950):
//   m = max_v x_v, s = sum_v e^(x_v - m), t = sum_v (x_v - m) e^(x_v - m)
//   logprob = (x_c - m) - ln s,   entropy = ln s - t / s,   alternatives: the largest x, ties to the lowest index
// A row's maximum and sums come from one pass: a running maximum rescales the sums (and t, whose terms all shift by the
// change of the maximum).

#include <math.h>

#include "common.h"

namespace mtl {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct LpArgs {
    const void* x;
    const int64_t* tokens;
    float* logprob;
    float* entropy;
    float* top_logprob;
    int64_t* top_token;
    int64_t inner, so, si;     // row i: x + (i / inner) so + (i % inner) si
    int V, top;
};

struct Sums {
    float m, s, t;             // s and t relative to max(m, lowest finite) ; m = -inf: nothing seen but -inf
};

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m), base = base_of(m);
    const float da = fmaxf(a.m - base, -1e30f), db = fmaxf(b.m - base, -1e30f);
    const float ea = fast_exp(da), eb = fast_exp(db);
    return {m, ea * a.s + eb * b.s, ea * fmaf(da, a.s, a.t) + eb * fmaf(db, b.s, b.t)};
}

// An order of (value, index): larger value first, then lower index.  0: no value (-inf never is an alternative).
__device__ __forceinline__ uint64_t key_of(float x, int i) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);     // -0 and 0 are equal
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return uint64_t(o) << 32 | uint32_t(~i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t o = uint32_t(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const LpArgs a) {
    __shared__ Sums s_sums[kWaves];
    __shared__ uint64_t s_key[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + (row / a.inner) * a.so + (row % a.inner) * a.si;

    Sums q = {-INFINITY, 0.f, 0.f};
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
        const float v = Act<T>::load(x + i);
        // (fmaxf drops a NaN; e^NaN reaches s all the same)
        const float m = fmaxf(q.m, v), base = base_of(m);
        if (m != q.m) {
            const float d = fmaxf(q.m - base, -1e30f), e = fast_exp(d);
            q = {m, e * q.s, e * fmaf(d, q.s, q.t)};
        }
        const float d = v - base, e = fast_exp(d);
        q.s += e;
        q.t = fmaf(fmaxf(d, -1e30f), e, q.t);
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) q = join(q, {__shfl_xor(q.m, o), __shfl_xor(q.s, o), __shfl_xor(q.t, o)});
    if (lane == 0) s_sums[wave] = q;
    __syncthreads();
    q = s_sums[0];
    for (int w = 1; w < kWaves; ++w) q = join(q, s_sums[w]);
    const float ls = logf(q.s);
    const bool empty = q.m == -INFINITY && q.s == 0.f, bad = !(fabsf(ls) < INFINITY) && !empty;
    if (threadIdx.x == 0) {
        const int64_t c = a.tokens[row];
        float lp = 0.f;
        if (c >= 0) lp = c >= a.V ? NAN : bad ? NAN : empty ? -INFINITY : (Act<T>::load(x + c) - q.m) - ls;
        a.logprob[row] = lp;
        a.entropy[row] = bad ? NAN : empty ? 0.f : ls - q.t / q.s;
    }
    uint64_t last = ~uint64_t(0);
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        if (!bad && last != 0)
            for (int i = threadIdx.x; i < a.V; i += kThreads) {
                const uint64_t key = key_of(Act<T>::load(x + i), i);
                if (key < last && key > best) best = key;
            }
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint64_t other = __shfl_xor((unsigned long long)best, o);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (lane == 0) s_key[wave] = best;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) best = s_key[w] > best ? s_key[w] : best;
        last = best;
        if (threadIdx.x == 0) {
            a.top_token[row * a.top + k] = best ? (int64_t)(uint32_t)~uint32_t(best) : -1;
            a.top_logprob[row * a.top + k] = bad ? NAN : best ? (key_value(best) - q.m) - ls : -INFINITY;
        }
    }
}

}  // namespace
}  // namespace mtl

extern "C" int mtl_token_logprobs(const mtl_token_logprobs_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    MTL_REQUIRE(p->dtype == MTL_F32 || p->dtype == MTL_BF16, "dtype must be MTL_F32 or MTL_BF16");
    MTL_REQUIRE(p->outer >= 0 && p->inner >= 0 && (p->inner == 0 || p->outer <= (int64_t(1) << 30) / p->inner),
                "at most 2^30 rows");
    MTL_REQUIRE(p->vocab >= 1 && p->vocab <= 1 << 30, "vocab must be in [1, 2^30]");
    MTL_REQUIRE(p->top >= 0 && p->top <= 64 && p->top <= p->vocab, "top must be in [0, min(64, vocab)]");
    if (p->outer * p->inner == 0) return MTL_OK;
    MTL_REQUIRE(p->logits && p->tokens && p->logprob && p->entropy && (p->top == 0 || (p->top_logprob && p->top_token)),
                "null pointer");
    const LpArgs a{p->logits, p->tokens, p->logprob, p->entropy, p->top_logprob, p->top_token, p->inner, p->stride_outer,
                   p->stride_inner, (int)p->vocab, p->top};
    const dim3 grid((unsigned)(p->outer * p->inner));
    if (p->dtype == MTL_F32) hipLaunchKernelGGL((logprob_kernel<float>), grid, dim3(kThreads), 0, as_stream(stream), a);
    else hipLaunchKernelGGL((logprob_kernel<uint16_t>), grid, dim3(kThreads), 0, as_stream(stream), a);
    return check_launch("token_logprobs");
}
