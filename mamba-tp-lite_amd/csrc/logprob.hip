// Log probabilities of given tokens, entropy and the most probable tokens of rows of logits (gfx950):
//   m = max_v x_v, s = sum_v e^(x_v - m), t = sum_v (x_v - m) e^(x_v - m)
//   logprob = (x_c - m) - ln s,   entropy = ln s - t / s,   alternatives: the largest x, ties to the lowest index
// A row's maximum and sums come from one pass: a running maximum rescales the sums (and t, whose terms all shift by the
// change of the maximum).

#include <float.h>
#include <math.h>

#include "common.h"

namespace mtl {
namespace {

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

__device__ __forceinline__ uint64_t lane_read64(uint64_t v, int lane) {
    return uint64_t(lane_read_u(uint32_t(v >> 32), lane)) << 32 | lane_read_u(uint32_t(v), lane);
}
__device__ __forceinline__ uint64_t xor_read64(uint64_t v, int m) {
    return uint64_t(uint32_t(__shfl_xor(int(v >> 32), m))) << 32 | uint32_t(__shfl_xor(int(v), m));
}

// The largest keys of what a wavefront has seen, one a lane in falling order; the first `top` lanes are right, the
// others hold further keys of it.
struct TopList {
    uint64_t key = 0, floor = 0;       // floor: the key of lane top - 1 (0: fewer seen), uniform
    float floor_value = -FLT_MAX;      // (above -inf, which never enters)

    __device__ __forceinline__ void set_floor(int top) {
        floor = lane_read64(key, top - 1);
        floor_value = floor ? key_value(floor) : -FLT_MAX;
    }
    // one lane's key each -> in falling order (bitonic)
    __device__ __forceinline__ void sort(uint64_t mine, int lane, int top) {
        key = mine;
#pragma unroll
        for (int size = 2; size <= 64; size *= 2)
#pragma unroll
            for (int m = size / 2; m > 0; m /= 2) {
                const uint64_t other = xor_read64(key, m);
                if ((other > key) == (((lane & m) == 0) == ((lane & size) == 0))) key = other;
            }
        set_floor(top);
    }
    // with another list in falling order: the larger of each and the reversed other are the 64 largest, bitonic
    __device__ __forceinline__ void merge(uint64_t other, int lane) {
        other = uint64_t(uint32_t(__shfl(int(other >> 32), 63 - lane))) << 32 | uint32_t(__shfl(int(other), 63 - lane));
        key = other > key ? other : key;
#pragma unroll
        for (int m = 32; m > 0; m /= 2) {
            const uint64_t x = xor_read64(key, m);
            if ((x > key) == ((lane & m) == 0)) key = x;
        }
    }
    // every lane's key above the floor, but `skip`
    __device__ __forceinline__ void insert(uint64_t mine, uint64_t skip, int lane, int top) {
        bool left = mine != skip;
        for (uint64_t mask; (mask = __ballot(left && mine > floor)) != 0;) {
            const int l = __builtin_ctzll(mask);
            const uint64_t c = lane_read64(mine, l);
            const int at = __builtin_popcountll(__ballot(key > c));
            const uint64_t up = uint64_t(uint32_t(__builtin_amdgcn_update_dpp(0, int(key >> 32), kDppWaveShr1, 0xF, 0xF, false))) << 32 |
                                uint32_t(__builtin_amdgcn_update_dpp(0, int(key), kDppWaveShr1, 0xF, 0xF, false));
            key = lane < at ? key : lane == at ? c : up;
            left = left && lane != l;
            set_floor(top);
        }
    }
};

// One workgroup per row, its wavefronts on tiles of 64 x kChunks 16-byte chunks in turn, the next tile in flight while
// one is summed.  A tile costs about ten instructions a logit; candidates for the list are looked for only where
// some lane's largest reaches the list's last value, which after the first tiles is rare.
constexpr int kChunks = 4, kTile = 64 * kChunks;
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

template <typename T, bool TOP>
__global__ void __launch_bounds__(1024) logprob_kernel(const LpArgs a) {
    constexpr int VEC = 16 / (int)sizeof(T);
    __shared__ Sums s_sums[16];
    __shared__ uint64_t s_list[TOP ? 16 : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + (row / a.inner) * a.so + (row % a.inner) * a.si;
    // chunk c holds logits c VEC - off .. + VEC - 1: chunks lie on 16-byte boundaries wherever the row starts
    const int off = int(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const int tiles = (int)(((int64_t)a.V + off + kTile * VEC - 1) / (kTile * VEC));

    U4 next[kChunks];
    auto load = [&](int tile) __attribute__((always_inline)) {
        const int64_t i0 = (int64_t)tile * kTile * VEC - off;
        if (i0 >= 0 && i0 + kTile * VEC <= a.V) {
#pragma unroll
            for (int u = 0; u < kChunks; ++u)
                next[u] = __builtin_nontemporal_load(reinterpret_cast<const U4*>(x + i0 + (u * 64 + lane) * VEC));
        } else {                                   // a row's ends: logit by logit, -inf outside
#pragma unroll
            for (int u = 0; u < kChunks; ++u) {
                T v[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int64_t i = i0 + (u * 64 + lane) * VEC + e;
                    if constexpr (sizeof(T) == 4) v[e] = i >= 0 && i < a.V ? x[i] : -INFINITY;
                    else v[e] = i >= 0 && i < a.V ? x[i] : T(0xff80);
                }
                __builtin_memcpy(&next[u], v, 16);
            }
        }
    };

    Sums q = {-INFINITY, 0.f, 0.f};
    TopList list;
    if (wave < tiles) load(wave);
    for (int tile = wave; tile < tiles; tile += waves) {
        float v[kChunks][VEC], most[kChunks];
#pragma unroll
        for (int u = 0; u < kChunks; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                v[u][e] = sizeof(T) == 4 ? __uint_as_float(next[u][e % 4])
                                         : __uint_as_float(e % 2 ? next[u][e / 2] & 0xffff0000u : next[u][e / 2] << 16);
        if (tile + waves < tiles) load(tile + waves);
        float m = q.m;
#pragma unroll
        for (int u = 0; u < kChunks; ++u) {
            most[u] = v[u][0];
#pragma unroll
            for (int e = 1; e < VEC; ++e) most[u] = fmaxf(most[u], v[u][e]);
            m = fmaxf(m, most[u]);
        }
        // (fmaxf drops a NaN; e^NaN reaches s all the same)
        const float base = base_of(m), d0 = fmaxf(q.m - base, -1e30f), e0 = fast_exp(d0);
        q = {m, e0 * q.s, e0 * fmaf(d0, q.s, q.t)};
#pragma unroll
        for (int u = 0; u < kChunks; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = v[u][e] - base, ex = fast_exp(d);
                q.s += ex;
                q.t = fmaf(fmaxf(d, -1e30f), ex, q.t);
            }
        if constexpr (TOP) {
            const int i0 = (int)((int64_t)tile * kTile * VEC - off) + lane * VEC;
            uint64_t mine = ~uint64_t(0);
            if (tile == wave) {                    // the first tile: the lanes' largest make the list
                mine = 0;
#pragma unroll
                for (int u = 0; u < kChunks; ++u)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const uint64_t k = key_of(v[u][e], i0 + u * 64 * VEC + e);
                        mine = k > mine ? k : mine;
                    }
                list.sort(mine, lane, a.top);
            }
#pragma unroll
            for (int u = 0; u < kChunks; ++u) {
                if (!__any(most[u] >= list.floor_value)) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (__any(v[u][e] >= list.floor_value))
                        list.insert(key_of(v[u][e], i0 + u * 64 * VEC + e), mine, lane, a.top);
            }
        }
    }

#pragma unroll
    for (int o = 1; o < 64; o *= 2) q = join(q, {__shfl_xor(q.m, o), __shfl_xor(q.s, o), __shfl_xor(q.t, o)});
    if (lane == 0) s_sums[wave] = q;
    if constexpr (TOP) s_list[wave][lane] = list.key;
    __syncthreads();
    if constexpr (TOP) {
        for (int h = 1; h < waves; h *= 2) {
            if (wave % (2 * h) == 0) {
                list.merge(s_list[wave + h][lane], lane);
                s_list[wave][lane] = list.key;
            }
            __syncthreads();
        }
    }
    if (wave != 0) return;
    for (int w = 1; w < waves; ++w) q = join(q, s_sums[w]);
    const float ls = logf(q.s);
    const bool empty = q.m == -INFINITY && q.s == 0.f, bad = !(fabsf(ls) < INFINITY) && !empty;
    if (lane == 0) {
        const int64_t c = a.tokens[row];
        float lp = 0.f;
        if (c >= 0) lp = c >= a.V || bad ? NAN : empty ? -INFINITY : (Act<T>::load(x + c) - q.m) - ls;
        a.logprob[row] = lp;
        a.entropy[row] = bad ? NAN : empty ? 0.f : ls - q.t / q.s;
    }
    if constexpr (TOP) {
        if (lane < a.top) {
            const uint64_t k = bad ? 0 : list.key;
            a.top_token[row * a.top + lane] = k ? (int64_t)(uint32_t)~uint32_t(k) : -1;
            a.top_logprob[row * a.top + lane] = bad ? NAN : k ? (key_value(k) - q.m) - ls : -INFINITY;
        }
    }
}

template <typename T>
int launch(const LpArgs& a, int64_t rows, hipStream_t st) {
    const int64_t tiles = (a.V + kTile * (16 / (int)sizeof(T)) - 1) / (kTile * (16 / (int)sizeof(T)));
    const int most = rows >= 2048 ? 4 : rows >= 512 ? 8 : 16;
    int waves = 1;
    while (waves < most && waves < tiles) waves *= 2;
    if (a.top) hipLaunchKernelGGL((logprob_kernel<T, true>), dim3((unsigned)rows), dim3(waves * 64), 0, st, a);
    else hipLaunchKernelGGL((logprob_kernel<T, false>), dim3((unsigned)rows), dim3(waves * 64), 0, st, a);
    return check_launch("token_logprobs");
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
    return p->dtype == MTL_F32 ? launch<float>(a, p->outer * p->inner, as_stream(stream))
                               : launch<uint16_t>(a, p->outer * p->inner, as_stream(stream));
}
