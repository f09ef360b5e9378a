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
    // how a row's floor is found, see launch()
    int shown, run_log2, share, again;
};

struct Sums {
    float m, s, t;             // s and t relative to max(m, lowest finite) ; m = -inf: nothing seen but -inf
};

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// a's sums relative to the maximum m >= a.m
__device__ __forceinline__ void rescale(Sums& a, float m) {
    const float d = fmaxf(a.m - base_of(m), -1e30f), e = fast_exp(d);
    a = {m, e * a.s, e * fmaf(d, a.s, a.t)};
}
// the sums of 16 or 64 lanes
template <int WIDTH>
__device__ __forceinline__ Sums group_join(Sums a) {
    rescale(a, group_max<WIDTH>(a.m));
    return {a.m, group_sum<WIDTH>(a.s), group_sum<WIDTH>(a.t)};
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
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_mov64(uint64_t v) {
    return uint64_t(dpp_mov_u<CTRL>(uint32_t(v >> 32))) << 32 | dpp_mov_u<CTRL>(uint32_t(v));
}
// the value of lane ^ M
template <int M>
__device__ __forceinline__ uint64_t xor_read64(uint64_t v) {
    constexpr int kQuadReverse = 0x1B, kRowRor8 = 0x128;
    if constexpr (M == 1) return dpp_mov64<kDppXor1>(v);
    else if constexpr (M == 2) return dpp_mov64<kDppXor2>(v);
    else if constexpr (M == 4) return dpp_mov64<kQuadReverse>(dpp_mov64<kDppHalfMirror>(v));     // 7 ^ 3
    else if constexpr (M == 8) return dpp_mov64<kRowRor8>(v);
    else return uint64_t(uint32_t(__shfl_xor(int(v >> 32), M))) << 32 | uint32_t(__shfl_xor(int(v), M));
}
// steps of a bitonic sort of the lanes in falling order: within runs of SIZE lanes, from distance M down
template <int SIZE, int M>
__device__ __forceinline__ void bitonic_steps(uint64_t& key, int lane) {
    const uint64_t other = xor_read64<M>(key);
    if ((other > key) == (((lane & M) == 0) == ((lane & SIZE) == 0))) key = other;
    if constexpr (M > 1) bitonic_steps<SIZE, M / 2>(key, lane);
}
template <int SIZE = 2>
__device__ __forceinline__ void bitonic_sort(uint64_t& key, int lane) {
    bitonic_steps<SIZE, SIZE / 2>(key, lane);
    if constexpr (SIZE < 64) bitonic_sort<SIZE * 2>(key, lane);
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    const uint32_t hi = group_umax<64>(uint32_t(v >> 32));
    return uint64_t(hi) << 32 | group_umax<64>(uint32_t(v >> 32) == hi ? uint32_t(v) : 0u);
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// place[o] += how many of this wavefront's share of n keys in LDS are larger than keys[o], for every o; zeros follow the
// keys (kPad of them)
constexpr int kPad = 8;
__device__ __forceinline__ void add_places(const uint64_t* keys, int n, int* place, int wave, int waves, int lane) {
    typedef uint64_t Pair __attribute__((ext_vector_type(2)));
    for (int o = lane; o < n; o += 64) {
        const uint64_t k = keys[o];
        int larger = 0;
        for (int i = wave * kPad; i < n; i += waves * kPad) {
            Pair other[kPad / 2];
#pragma unroll
            for (int e = 0; e < kPad / 2; ++e) other[e] = *reinterpret_cast<const Pair*>(keys + i + 2 * e);
#pragma unroll
            for (int e = 0; e < kPad; ++e) larger += other[e / 2][e % 2] > k;
        }
        if (larger) atomicAdd(&place[o], larger);
    }
}

// Candidates of one wavefront for the row's `top` largest keys: those that reach the floor, a key that `top` keys of
// the row are known to reach.  They wait in LDS (64 to a flush); a flush merges them into a sorted list of 64, one a
// lane, whose last wanted key is a floor too.
struct Candidates {
    uint64_t* wait;                    // [128]
    uint64_t* shared;                  // the highest floor a flush of any wavefront has found
    uint64_t list = 0, floor = 1;
    float floor_value = -FLT_MAX;      // (above -inf, which never enters)
    int waiting = 0;

    __device__ __forceinline__ void raise(uint64_t f) {
        if (f > floor) {
            floor = f;
            floor_value = key_value(f);
        }
    }
    __device__ __forceinline__ void see() {
        raise(lane_read64(__hip_atomic_load(shared, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP), 0));
    }
    __device__ __forceinline__ void add(uint64_t key, int lane, int top) {
        const bool hit = key >= floor;
        const uint64_t mask = __ballot(hit);
        if (hit) wait[waiting + __builtin_popcountll(mask & ((uint64_t(1) << lane) - 1))] = key;
        waiting += __builtin_popcountll(mask);
        if (waiting >= 64) flush(lane, top);
    }
    __device__ __forceinline__ void flush(int lane, int top) {
        wave_lds_fence();
        uint64_t k = lane < waiting ? wait[lane] : 0;
        bitonic_sort(k, lane);
        // the larger of each and the reversed other list are the 64 largest, in bitonic order
        k = uint64_t(uint32_t(__shfl(int(k >> 32), 63 - lane))) << 32 | uint32_t(__shfl(int(k), 63 - lane));
        list = k > list ? k : list;
        bitonic_steps<64, 32>(list, lane);
        k = wait[64 + lane];
        waiting = max(waiting - 64, 0);
        wave_lds_fence();
        if (lane < waiting) wait[lane] = k;
        const uint64_t f = lane_read64(list, top - 1);
        raise(f);
        if (lane == 0) __hip_atomic_fetch_max(shared, f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        see();
    }
};

// One workgroup per row, its wavefronts on tiles of 64 x kChunks 16-byte chunks in turn, the next tile in flight while
// one is summed.  A tile costs about ten instructions a logit; candidates for the list are looked for only where
// some lane's largest reaches the list's last value, which after the first tiles is rare.
constexpr int kChunks = 4, kTile = 64 * kChunks;
constexpr int kShown = 256;            // 16 of each of 16 wavefronts
constexpr int kKeptBytes = 2 * sizeof(uint64_t) + sizeof(int);
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

template <typename T, bool TOP>
__global__ void __launch_bounds__(1024) logprob_kernel(const LpArgs a) {
    constexpr int VEC = 16 / (int)sizeof(T);
    __shared__ Sums s_sums[16];
    __shared__ __align__(16) uint64_t s_shown[TOP ? kShown + kPad : 1], s_least[16], s_again[16];
    __shared__ int s_keys, s_shown_place[TOP ? kShown : 1];
    __shared__ uint64_t s_floor;
    extern __shared__ __align__(16) uint64_t s_key[];      // TOP: [waves][128] waiting, [waves][128] kept, their places
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t row = blockIdx.x;
    const uint32_t outer = blockIdx.x / (uint32_t)a.inner;     // (fewer than 2^24 rows)
    const T* x = static_cast<const T*>(a.x) + outer * a.so + (blockIdx.x - outer * (uint32_t)a.inner) * a.si;
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

    if (wave < tiles) load(wave);
    __builtin_amdgcn_sched_barrier(0);
    int64_t token = 0;
    float given = 0.f;                              // the token's logit
    if (threadIdx.x == 0) {
        s_keys = 0;
        s_floor = 0;
        token = a.tokens[row];
        if (token >= 0 && token < a.V) given = Act<T>::load(x + token);
    }
    Sums q = {-INFINITY, 0.f, 0.f};
    Candidates c;
    c.wait = s_key + wave * 128;
    c.shared = &s_floor;
    uint64_t* keep = s_key + waves * 128;
    int* place = reinterpret_cast<int*>(keep + waves * 128 + kPad);
    if constexpr (TOP) {
        typedef uint64_t Pair __attribute__((ext_vector_type(2)));
        reinterpret_cast<Pair*>(keep)[threadIdx.x] = Pair{0, 0};
        reinterpret_cast<uint64_t*>(place)[threadIdx.x] = 0;
        if (threadIdx.x < a.shown) s_shown_place[threadIdx.x] = 0;
        if (threadIdx.x < kPad) keep[waves * 128 + threadIdx.x] = s_shown[a.shown + threadIdx.x] = 0;
    }
    auto least = [&](const uint64_t* of) __attribute__((always_inline)) { return ~wave_max64(~of[min(lane, waves - 1)]); };
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
        rescale(q, m);
        const float base = base_of(m);
        // (a tile's terms by themselves first: one rounding a tile, not one a term, falls on the running sums, which the
        // row's few large terms have made large)
        float s[kChunks], t[kChunks];
#pragma unroll
        for (int u = 0; u < kChunks; ++u) {
            s[u] = t[u] = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = v[u][e] - base, ex = fast_exp(d);
                s[u] += ex;
                t[u] = fmaf(fmaxf(d, -1e30f), ex, t[u]);
            }
        }
        static_assert(kChunks == 4, "four partial sums");
        q.s += (s[0] + s[1]) + (s[2] + s[3]);
        q.t += (t[0] + t[1]) + (t[2] + t[3]);
        if constexpr (TOP) {
            const int i0 = (int)((int64_t)tile * kTile * VEC - off) + lane * VEC;
            float all = most[0];
#pragma unroll
            for (int u = 1; u < kChunks; ++u) all = fmaxf(all, most[u]);
            if (tile == wave) {
                // the first tile sets the floor
                int at = 0;                        // the lowest index of the lane's largest
#pragma unroll
                for (int n = kChunks * VEC - 1; n > 0; --n) at = v[n / VEC][n % VEC] == all ? n / VEC * 64 * VEC + n % VEC : at;
                uint64_t k = key_of(all, i0 + (v[0][0] == all ? 0 : at));
                if (a.share >= 0) {
                    bitonic_sort(k, lane);
                    if (lane == a.share) s_least[wave] = k;
                    lds_barrier();
                    c.raise(least(s_least));
                } else {
                    if (a.run_log2 == 6) {
                        k = wave_max64(k);
                    } else {
                        k = max64(k, dpp_mov64<kDppXor1>(k));
                        k = max64(k, dpp_mov64<kDppXor2>(k));
                        if (a.run_log2 > 2) k = max64(k, dpp_mov64<kDppHalfMirror>(k));
                        if (a.run_log2 > 3) k = max64(k, dpp_mov64<kDppRowMirror>(k));
                    }
                    if ((lane & ((1 << a.run_log2) - 1)) == 0) s_shown[(wave * 64 + lane) >> a.run_log2] = k;
                    lds_barrier();
                    add_places(s_shown, a.shown, s_shown_place, wave, waves, lane);
                    lds_barrier();
                    for (int o0 = 0; o0 < a.shown; o0 += 64) {
                        const int o = min(o0 + lane, a.shown - 1);
                        const uint64_t mask = __ballot(s_shown_place[o] == a.top - 1);
                        if (mask) c.raise(lane_read64(s_shown[o], __builtin_ctzll(mask)));
                    }
                }
            }
            if (__any(all >= c.floor_value)) {
#pragma unroll
                for (int u = 0; u < kChunks; ++u) {
                    if (!__any(most[u] >= c.floor_value)) continue;
                    // which of a lane's logits reach the floor; they enter one a lane at a time
                    uint32_t which = 0;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) which |= (v[u][e] >= c.floor_value ? 1u : 0u) << e;
                    while (__any(which != 0)) {
                        const int e = __builtin_ctz(which | 1u << (VEC - 1));
                        float value = v[u][0];
#pragma unroll
                        for (int n = 1; n < VEC; ++n) value = e == n ? v[u][n] : value;
                        const uint64_t k = which ? key_of(value, i0 + u * 64 * VEC + e) : 0;
                        c.add(k, lane, a.top);
                        which &= which - 1;
                    }
                }
            }
        }
    }

    q = group_join<64>(q);
    if (lane == 0) s_sums[wave] = q;
    if constexpr (TOP) {
        // What reaches the floor is little more than `top` keys.  They are put side by side in any order; a key's place in
        // the answer is how many are larger.
        if (a.again >= 0) {
            if (c.waiting) c.flush(lane, a.top);
            if (lane == a.again) s_again[wave] = c.list;
            lds_barrier();
            c.raise(least(s_again));
        }
        c.see();
        const uint64_t k0 = lane < a.top ? c.list : 0, k1 = lane < c.waiting ? c.wait[lane] : 0;
        const uint64_t mask0 = __ballot(k0 >= c.floor), mask1 = __ballot(k1 >= c.floor);
        const int n0 = __builtin_popcountll(mask0), n1 = __builtin_popcountll(mask1);
        int first = 0;
        if (lane == 0 && n0 + n1) first = atomicAdd(&s_keys, n0 + n1);
        first = __builtin_amdgcn_readfirstlane(first);
        const uint64_t below = (uint64_t(1) << lane) - 1;
        if (mask0 >> lane & 1) keep[first + __builtin_popcountll(mask0 & below)] = k0;
        if (mask1 >> lane & 1) keep[first + n0 + __builtin_popcountll(mask1 & below)] = k1;
    }
    lds_barrier();
    q = (lane & 15) < waves ? s_sums[lane & 15] : Sums{-INFINITY, 0.f, 0.f};
    q = group_join<16>(q);
    // one lane's (a product fused into a sum of two lanes rounds differently in the two)
    q = {lane_read(q.m, 0), lane_read(q.s, 0), lane_read(q.t, 0)};
    const float ls = logf(q.s);
    const bool empty = q.m == -INFINITY && q.s == 0.f, bad = !(fabsf(ls) < INFINITY) && !empty;
    if (threadIdx.x == 0) {
        float lp = 0.f;
        if (token >= 0) lp = token >= a.V || bad ? NAN : empty ? -INFINITY : (given - q.m) - ls;
        a.logprob[row] = lp;
        a.entropy[row] = bad ? NAN : empty ? 0.f : ls - q.t / q.s;
    }
    if constexpr (TOP) {
        const int keys = bad ? 0 : s_keys;
        add_places(keep, keys, place, wave, waves, lane);
        lds_barrier();
        for (int o = threadIdx.x; o < keys; o += blockDim.x) {
            const int at = place[o];
            if ((uint32_t)at < (uint32_t)a.top) {
                const uint64_t k = keep[o];
                a.top_token[row * a.top + at] = (int64_t)(uint32_t)~uint32_t(k);
                a.top_logprob[row * a.top + at] = (key_value(k) - q.m) - ls;
            }
        }
        if (wave == 0 && lane >= keys && lane < a.top) {         // fewer than `top` tokens are left
            a.top_token[row * a.top + lane] = -1;
            a.top_logprob[row * a.top + lane] = bad ? NAN : -INFINITY;
        }
    }
}

template <typename T>
int launch(LpArgs a, int64_t rows, hipStream_t st) {
    const int64_t tiles = (a.V + kTile * (16 / (int)sizeof(T)) - 1) / (kTile * (16 / (int)sizeof(T)));
    // Few rows: many wavefronts each, past 256 no more than two rows on a CU leave room for; no more than share the tiles
    // evenly, and every one has a first tile (the kernel's barrier after it counts on that).  Rows of 50280 with 5
    // alternatives, us: 300 fp32 with 8 wavefronts 17.9, 13 21.7; 513 bf16 with 7 23.6, 5 26.7; 1022 bf16 with 4 31.3,
    // 8 32.8, 16 44.7.
    const int64_t most = std::clamp<int64_t>(4096 / rows, 4, rows <= 256 ? 16 : 8), turns = (tiles + most - 1) / most;
    const int waves = (int)((tiles + turns - 1) / turns);
    // The floor from the first tiles: each wavefront shows the largest key of every run of lanes, the longest runs (64, 16, 8
    // or 4 lanes) that make 2 top of them, and the top-th largest of those is the floor.  Where runs of 4 are too few, the
    // wavefronts sort their lanes' and the least of their (top / wavefronts)-th is not far below.  Then about
    // top x tiles / wavefronts keys reach it, and where counting all of those would take longer than a sort in each wavefront,
    // a second floor comes from the wavefronts' sorted lists.  Measured, us, against floors from the least of the wavefronts'
    // last shown throughout: 32 rows of 50280 with 20 alternatives 12.3, 15.7; 256 of 6285 with 20 6.9, 14.2; 37 of 10007
    // with 64 8.6, 11.7; 1 of 50280 with 5 10.0, 10.7; and 300 of 2100 with 64, where they still sort, 20.5, 22.7.
    const int share = (a.top - 1) / waves;
    a.run_log2 = 6;
    while (waves << (6 - a.run_log2) < 2 * a.top && a.run_log2 > 2) a.run_log2 -= a.run_log2 == 6 ? 2 : 1;
    a.shown = waves << (6 - a.run_log2);
    a.share = a.shown < 2 * a.top ? share : -1;
    const int64_t keys = a.top * tiles / waves;
    a.again = waves > 1 && tiles > waves && keys * keys > 1024 * waves ? share : -1;
    if (a.top) {
        const size_t lds = waves * 128 * kKeptBytes + kPad * sizeof(uint64_t);
        hipLaunchKernelGGL((logprob_kernel<T, true>), dim3((unsigned)rows), dim3(waves * 64), lds, st, a);
    }
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
    // (a launch holds fewer than 2^32 threads, of which a row takes up to 256 where there are many)
    MTL_REQUIRE(p->outer >= 0 && p->inner >= 0 && (p->inner == 0 || p->outer <= ((int64_t(1) << 24) - 1) / p->inner),
                "at most 2^24 - 1 rows");
    MTL_REQUIRE(p->vocab >= 1 && p->vocab <= 1 << 30, "vocab must be in [1, 2^30]");
    MTL_REQUIRE(p->top >= 0 && p->top <= 64 && p->top <= p->vocab, "top must be in [0, min(64, vocab)]");
    if (p->outer * p->inner == 0) return MTL_OK;
    MTL_REQUIRE(p->logits && p->tokens && p->logprob && p->entropy && (p->top == 0 || (p->top_logprob && p->top_token)),
                "null pointer");
    const LpArgs a{p->logits, p->tokens, p->logprob, p->entropy, p->top_logprob, p->top_token, p->inner, p->stride_outer,
                   p->stride_inner, (int)p->vocab, p->top, 0, 0, -1, -1};
    return p->dtype == MTL_F32 ? launch<float>(a, p->outer * p->inner, as_stream(stream))
                               : launch<uint16_t>(a, p->outer * p->inner, as_stream(stream));
}
