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
    int y_f32;                 // y holds floats whatever x is
};

// the code of column 32 i + 8 j + e in word w
__device__ __forceinline__ uint32_t code_of(uint32_t w, int e) { return (w >> (16 * (e & 1) + 4 * (e >> 1))) & 15u; }

template <typename S> __device__ __forceinline__ float scale_at(const void* p, int64_t i) {
    if constexpr (sizeof(S) == 2) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}

typedef __bf16 B8h __attribute__((ext_vector_type(8)));
typedef uint16_t H2 __attribute__((ext_vector_type(2)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

// The weights of a word's 8 codes, in order, as bf16 numbers in units of kUnit: with zeros (z in every byte) q - z through
// the signed bytes of a register (19 instructions), without them (q - 8) / 16 of the nibbles q ^ 8, two's complements,
// which one conversion makes (14).
template <bool Z> constexpr float kUnit = Z ? 1.f : 0.0625f;
template <bool Z> __device__ __forceinline__ B8h word_weights(uint32_t c, uint32_t zeros) {
    float f[8];
    if constexpr (Z) {
        // q + 128 - z in every byte: no borrow leaves it
        const uint32_t lo = (((c & 0x0f0f0f0fu) | 0x80808080u) - zeros) ^ 0x80808080u;
        const uint32_t hi = (((c >> 4 & 0x0f0f0f0fu) | 0x80808080u) - zeros) ^ 0x80808080u;
#pragma unroll
        for (int b = 0; b < 4; ++b) {              // byte b: codes (b / 2) + 4 (b & 1) and 2 more
            f[b / 2 + 4 * (b & 1)] = (float)(int8_t)(lo >> (8 * b));
            f[b / 2 + 4 * (b & 1) + 2] = (float)(int8_t)(hi >> (8 * b));
        }
    } else {
        const uint32_t lo = c ^ 0x88888888u;
        uint32_t hi = lo >> 4;
        asm("" : "+v"(hi));                        // (its bytes are operands then, not shifts of lo)
#pragma unroll
        for (int b = 0; b < 4; ++b) {              // (the conversion reads four bits)
            f[b / 2 + 4 * (b & 1)] = __builtin_amdgcn_cvt_off_f32_i4(b ? lo >> (8 * b) & 0xffu : lo);
            f[b / 2 + 4 * (b & 1) + 2] = __builtin_amdgcn_cvt_off_f32_i4(b ? hi >> (8 * b) & 0xffu : hi);
        }
    }
    U4 pairs;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        pairs[i] = __builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302);
    return __builtin_bit_cast(B8h, pairs);
}

constexpr int kWaves = 16;                 // most wavefronts of a workgroup
constexpr uint32_t kWide = 0x6f800000u;    // 2^96
constexpr int kAhead = 4;                  // blocks of W that a wavefront has in flight
constexpr int kLdsBytes = 158 << 10;

struct LinearW4 {
    W4Args a;
    int rows;                  // rows of x per workgroup (blockIdx.y takes the next ones)
    int kblocks;               // 128-column blocks of x in LDS at a time
    int wk, wk_log2;           // wavefronts that share a tile of W, each on every wk-th block
};

template <typename S, int NG> struct alignas(sizeof(S) * NG) Scales {        // one row's scales of a block
    S v[NG];
    __device__ __forceinline__ float at(int g) const {
        if constexpr (sizeof(S) == 2) return bf16_to_f32(v[g]);
        else return v[g];
    }
};

// Products on the bf16 matrix cores, exact: q - z is a bf16 number, x in float32 the sum of three bf16 numbers of 8
// significand bits each (down to bf16's least, 2^-133), as rows of their own.  A group's sums run in fp32 on
// v_mfma_f32_16x16x32_bf16:
//   acc += s sum x (q - z)
// (Products with 16 + q, which the four bits under an exponent give for half the instructions, less x times 16 + z leave
// the rounding of sums of 31 |x|, on columns of zero weight too.)
//
// A workgroup keeps x, as the operand's 16-byte runs, in LDS; each wavefront streams tiles of W into registers, kAhead
// blocks before their use.  Where there are few tiles, wk wavefronts share one and add their sums in order.
//
// |x| >= 2^96 could overflow before its scale is applied, and infinities and NaN have no three parts: a row that holds one
// in a part of x is zeros there to the matrix cores, and takes its products weight by weight, as the matrix form would
// round them.  Other rows stay as they are, to the bit.
template <typename T, typename S, int G, bool Z, int TM>
__global__ void __launch_bounds__(kWaves * 64) linear_w4_kernel(const LinearW4 p) {
    constexpr int NG = kBlockK / G, P = sizeof(T) == 4 ? 3 : 1, R16 = TM * 16;
    extern __shared__ __align__(16) uint8_t smem[];
    const W4Args& a = p.a;
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m0 = blockIdx.y * p.rows, M = min(p.rows, a.M - m0), R = P * M;
    const int threads = blockDim.x, wn = wave >> p.wk_log2, wkid = wave & (p.wk - 1), WN = threads / 64 >> p.wk_log2;
    const T* x = static_cast<const T*>(a.x) + m0 * a.ldx;
    const int pitch = p.kblocks * 16 + 1;                     // (+ 1: the 16 rows of an operand start in different banks)
    U4* s_x = reinterpret_cast<U4*>(smem);                    // [R][k / 8]
    int at_x[TM];
#pragma unroll
    for (int q = 0; q < TM; ++q) at_x[q] = min(q * 16 + r, R - 1) * pitch + j;
    float* s_red = reinterpret_cast<float*>(s_x + P * p.rows * pitch);                         // [wave][R16][16]
    __shared__ uint32_t s_wide;                               // bit m: row m of this part of x is such a one

    // u / n8 for the fewer than 2^19 runs of x and at most 48 rows: the product is off by less than half of 1 / n8
    auto row_of = [&](int u, float inv) __attribute__((always_inline)) { return (int)((u + 0.5f) * inv); };
    // x to LDS: a thread takes 8 columns of a row at a time, kUnits of them in flight (8 of bf16 spill beside two operand
    // tiles).  Whole runs at any alignment: rows of 777 bf16 taken value by value where they start off a 16-byte boundary
    // cost 1.3 of 6.4 us at 33 rows for 1001 rows of W.
    constexpr int kRaw = 8 * (int)sizeof(T) / 16, kUnits = P > 1 ? 2 : TM == 1 ? 8 : 4;
    U4 raw[kUnits][kRaw];
    auto fetch = [&](int kb0, int nb, int u0) __attribute__((always_inline)) {
        const int n8 = nb * 16, runs = a.K < 8 ? 0 : M * n8;
        const float inv = 1.f / n8;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            if (__builtin_amdgcn_readfirstlane(u0) + n * threads >= runs) break;
            const int u = min(u0 + n * threads, runs - 1), m = row_of(u, inv), k = kb0 * kBlockK + (u - m * n8) * 8;
            // (the row's last 8 again where fewer are left: put_end shifts them)
            __builtin_memcpy(raw[n], x + m * a.ldx + min(k, a.K - 8), sizeof(raw[n]));
        }
    };
    auto put = [&](int nb, int u0) __attribute__((always_inline)) {
        const int n8 = nb * 16, runs = a.K < 8 ? 0 : M * n8;
        const float inv = 1.f / n8;
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            const int u = u0 + n * threads;
            if (u >= runs) break;
            const int m = row_of(u, inv), k8 = u - m * n8;
            if constexpr (P == 1) {                // bf16 as it is; its largest magnitude two values at a time
                H2 most = {0, 0};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    most = __builtin_elementwise_max(most, __builtin_bit_cast(H2, raw[n][0][q] & 0x7fff7fffu));
                if (max(most[0], most[1]) >= (kWide >> 16)) atomicOr(&s_wide, 1u << m);
                s_x[m * pitch + k8] = raw[n][0];
            } else {
                float v[8];
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = __uint_as_float(raw[n][e / 4 % kRaw][e % 4]);
                    most = max(most, abs_bits(v[e]));
                }
                if (most >= kWide) atomicOr(&s_wide, 1u << m);
#pragma unroll
                for (int q = 0; q < P; ++q) {      // the upper 8 significand bits of what is left, three times
                    U4 part;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        part[e / 2] = __builtin_amdgcn_perm(__float_as_uint(v[e + 1]), __float_as_uint(v[e]), 0x07060302);
                        v[e] -= __uint_as_float(__float_as_uint(v[e]) & 0xffff0000u);
                        v[e + 1] -= __uint_as_float(__float_as_uint(v[e + 1]) & 0xffff0000u);
                    }
                    s_x[(q * M + m) * pitch + k8] = part;
                }
            }
        }
    };

    // the last block's runs that reach past the row: the row's last 8 values, which are there, shifted down, zeros behind
    auto put_end = [&](int kb0) __attribute__((always_inline)) {
        for (int u = threadIdx.x; u < M * 16; u += threads) {
            const int m = u >> 4, k = (a.KB - 1) * kBlockK + (u & 15) * 8, past = k + 8 - a.K;
            if (past <= 0) continue;
            uint16_t* run = reinterpret_cast<uint16_t*>(s_x + m * pitch) + k - kb0 * kBlockK;
            if (a.K < 8) {                         // (nothing is there)
#pragma unroll 1
                for (int e = 0; e < 8; ++e) {
                    float v = k + e < a.K ? Act<T>::load(x + m * a.ldx + k + e) : 0.f;
                    if (abs_bits(v) >= kWide) atomicOr(&s_wide, 1u << m);
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        run[q * M * pitch * 8 + e] = __float_as_uint(v) >> 16;
                        v -= __uint_as_float(__float_as_uint(v) & 0xffff0000u);
                    }
                }
                continue;
            }
#pragma unroll
            for (int q = 0; q < P; ++q) {
                uint16_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = run[q * M * pitch * 8 + min(e + past, 7)];
#pragma unroll
                for (int e = 0; e < 8; ++e) run[q * M * pitch * 8 + e] = e + past < 8 ? v[e] : 0;
            }
        }
    };

    const int tiles = (a.N + kTileRows - 1) / kTileRows;
    const bool once = p.kblocks >= a.KB;

    // kAhead blocks of W in registers; as one is used up, the block kAhead further on (of the next tile, after the
    // last) is loaded in its place, so the stream never stops at the end of a tile.  The loads stand in no branch: the
    // wait before a block's use then counts the younger ones out.
    U4 w[kAhead];
    Scales<S, NG> sc[kAhead];
    Scales<uint8_t, NG> zr[kAhead];
    auto load = [&](int u, int64_t b0, int last) __attribute__((always_inline)) {
        const int64_t b = b0 + min(u, last) * p.wk;          // (a batch's last block again, past it)
        w[u] = __builtin_nontemporal_load(reinterpret_cast<const U4*>(a.codes) + b * 64 + lane);
        sc[u] = static_cast<const Scales<S, NG>*>(a.scales)[b * kTileRows + r];
        if constexpr (Z) zr[u] = reinterpret_cast<const Scales<uint8_t, NG>*>(a.zeros)[b * kTileRows + r];
    };
    F4v acc[TM];
    // acc += the block in slot u times columns 128 kc .. of the part of x in LDS
    auto multiply = [&](int u, int kc) __attribute__((always_inline)) {
        F4v part[TM];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i % (G / 32) == 0) {
#pragma unroll
                for (int q = 0; q < TM; ++q) part[q] = F4v{0.f, 0.f, 0.f, 0.f};
            }
            // (x on its way while the codes are unpacked: 16 rows by 50280 x 2048 17.5 us, read after it 18.4)
            B8h xa[TM];
#pragma unroll
            for (int q = 0; q < TM; ++q) xa[q] = __builtin_bit_cast(B8h, s_x[at_x[q] + kc * 16 + i * 4]);
            __builtin_amdgcn_sched_barrier(0);
            uint32_t zeros = 0;                    // the group's, in every byte
            if constexpr (Z) {
                __builtin_memcpy(&zeros, &zr[u], NG);
                zeros = __builtin_amdgcn_perm(0u, zeros, 0x01010101u * (i / (G / 32)));
            }
            const B8h weights = word_weights<Z>(w[u][i], zeros);
#pragma unroll
            for (int q = 0; q < TM; ++q)
                part[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa[q], weights, part[q], 0, 0, 0);
            if (i % (G / 32) == G / 32 - 1) {
                const float s = sc[u].at(i / (G / 32));
#pragma unroll
                for (int q = 0; q < TM; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[q][e] = fmaf(s, part[q][e], acc[q][e]);
            }
        }
    };
    const int stride = gridDim.x * WN;
    int t = blockIdx.x * WN + wn;
    // (x before W: what waits for x then does not wait for W, whose loads return after it)
    fetch(0, min(p.kblocks, a.KB), threadIdx.x);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) load(u, (int64_t)min(t, tiles - 1) * a.KB + wkid, (a.KB - 1 - wkid) >> p.wk_log2);
    __builtin_amdgcn_sched_barrier(0);
    if (threadIdx.x == 0) s_wide = 0;
    lds_barrier();
    put(min(p.kblocks, a.KB), threadIdx.x);                  // (here, not in the loop: its wait then counts W's loads out)
    int u0 = threadIdx.x + kUnits * threads;                 // the first run of x that is not in LDS yet
    bool staged = false;
    for (int t0 = blockIdx.x * WN; t0 < tiles; t0 += stride, t += stride) {
#pragma unroll
        for (int q = 0; q < TM; ++q) acc[q] = F4v{0.f, 0.f, 0.f, 0.f};
        for (int kb0 = 0; kb0 < a.KB; kb0 += p.kblocks) {
            const int kb1 = min(kb0 + p.kblocks, a.KB);
            if (!once || !staged) {
                const int nb = kb1 - kb0;
                if (staged) {
                    lds_barrier();
                    if (threadIdx.x == 0) s_wide = 0;
                    lds_barrier();
                    u0 = threadIdx.x;
                }
                for (; u0 < M * nb * 16; u0 += kUnits * threads) {
                    fetch(kb0, nb, u0);
                    put(nb, u0);
                }
                if (a.K % kBlockK != 0 && kb1 == a.KB) {
                    lds_barrier();
                    put_end(kb0);
                }
                staged = true;
                lds_barrier();
                if (s_wide) {
                    for (int u = threadIdx.x; u < R * nb * 16; u += threads) {
                        const int row = u / (nb * 16);
                        if (s_wide >> row % M & 1) s_x[row * pitch + u - row * nb * 16] = U4{0, 0, 0, 0};
                    }
                    lds_barrier();
                }
            }
            uint32_t wide = __builtin_amdgcn_readfirstlane(s_wide);
            for (int kb = kb0 + wkid; kb < kb1; kb += kAhead * p.wk) {
                const bool more = kb + kAhead * p.wk < a.KB;
                const int tn = more ? t : t + stride, kbn = more ? kb + kAhead * p.wk : wkid;
                const int blocks = ((kb1 - 1 - kb) >> p.wk_log2) + 1, kc = kb - kb0;
                if (tn < tiles) {
                    const int64_t b0 = (int64_t)tn * a.KB + kbn;
                    const int last = (a.KB - 1 - kbn) >> p.wk_log2;
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        if (u < blocks) multiply(u, kc + u * p.wk);
                        load(u, b0, last);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < kAhead; ++u)
                        if (u < blocks) multiply(u, kc + u * p.wk);
                }
            }
            const int64_t tb = (int64_t)min(t, tiles - 1) * a.KB;
            for (; wide; wide &= wide - 1) {
                const int m = __builtin_ctz(wide);
                float v = 0.f;
#pragma unroll 1
                for (int kb = kb0 + wkid; kb < kb1; kb += p.wk) {
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t c = reinterpret_cast<const uint32_t*>(a.codes)[((tb + kb) * 64 + lane) * 4 + i];
                        const int64_t at = ((tb + kb) * kTileRows + r) * NG + 32 * i / G;
                        const float s = scale_at<S>(a.scales, at), z = Z ? (float)a.zeros[at] : 8.f;
                        const int k = kb * kBlockK + 32 * i + 8 * j;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (k + e < a.K) v = fmaf(Act<T>::load(x + m * a.ldx + k + e), s * ((float)code_of(c, e) - z), v);
                    }
                }
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                // into row m's accumulator: lanes 4 j .. + 3 of tile m / 16
#pragma unroll
                for (int q = 0; q < TM * 4; ++q)
                    if ((m >> 4) * 4 + (m & 3) == q && ((m >> 2) & 3) == j) acc[q >> 2][q & 3] += v * kUnit<Z>;
            }
        }
        // D[i][j]: row 4 (lane / 16) + i of x, row lane % 16 of W
#pragma unroll
        for (int q = 0; q < TM; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) s_red[(wave * R16 + q * 16 + 4 * j + e) * 16 + r] = acc[q][e];
        // a quarter of a wavefront to a row m of a tile; where a sum has many parts all four to one, a fourth each
        const int parts = P * p.wk;
        const bool spread = parts >= 8;
        auto store = [&](int tile, int first, int m) __attribute__((always_inline)) {
            float v = 0.f;
#pragma unroll 4
            for (int i = spread ? j : 0; i < parts; i += spread ? 4 : 1)
                v += s_red[((first + (i & (p.wk - 1))) * R16 + (i >> p.wk_log2) * M + m) * 16 + r];
            if (spread) {
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
            }
            v *= 1.f / kUnit<Z>;
            const int n = tile * kTileRows + r;
            if ((j == 0 || !spread) && n < a.N) {
                if (a.bias) v += Act<T>::load(static_cast<const T*>(a.bias) + n);
                const int64_t at = (m0 + m) * a.ldy + n;
                if (a.y_f32) static_cast<float*>(a.y)[at] = v;
                else Act<T>::store(static_cast<T*>(a.y) + at, v);
            }
        };
        if (p.wk == 1) {                                     // a wavefront's own sums: no other waits for it
            wave_lds_fence();
            for (int m = j; m < M; m += 4) store(t, wave, m);
            wave_lds_fence();
        } else {
            lds_barrier();
            const int step = threads / (spread ? 64 : 16);
            for (int mt = spread ? wave : (int)threadIdx.x >> 4; mt < WN * M; mt += step) {
                const int ti = WN == 1 ? 0 : mt / M;
                store(t0 + ti, ti * p.wk, mt - ti * M);
            }
            lds_barrier();
        }
    }
}

// One wavefront per tile of 16 rows x 128 columns, through LDS, so that a store writes neighbouring columns of a row or
// a few whole rows: with rows of W on 16-byte boundaries (VEC) 16 bytes a lane, else a value.  (Lanes that stored their
// own 8 columns, 64-byte pieces of 16 rows at a time, took 61 us for 24323 x 3784 bf16, 3.8 TB/s.)
template <typename T, typename S, int G, bool Z, bool VEC>
__global__ void __launch_bounds__(256) dequantize_w4_kernel(const W4Args a) {
    constexpr int NG = kBlockK / G;
    constexpr int kPer = 16 / (int)sizeof(T), kPitch = kBlockK + kPer;       // (rows start in different banks)
    __shared__ __align__(16) T s_row[4][kTileRows * kPitch];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, j = lane >> 4;
    const int64_t tile = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + wave, t = tile / a.KB;
    const int kb = (int)(tile - t * a.KB);
    const int64_t n0 = t * kTileRows;
    if (n0 >= a.N) return;
    const int64_t b = t * a.KB + kb;
    const U4 w = __builtin_nontemporal_load(reinterpret_cast<const U4*>(a.codes) + b * 64 + lane);
    const Scales<S, NG> sc = static_cast<const Scales<S, NG>*>(a.scales)[b * kTileRows + r];
    Scales<uint8_t, NG> zr;
    if constexpr (Z) zr = reinterpret_cast<const Scales<uint8_t, NG>*>(a.zeros)[b * kTileRows + r];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s = sc.at(i / (G / 32));
        const int zero = Z ? zr.v[i / (G / 32)] : 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s * (float)((int)code_of(w[i], e) - zero);
        T* to = &s_row[wave][r * kPitch + 32 * i + 8 * j];
        if constexpr (sizeof(T) == 4) {
            st4(to, F4v{v[0], v[1], v[2], v[3]});
            st4(to + 4, F4v{v[4], v[5], v[6], v[7]});
        } else {
            *reinterpret_cast<U4*>(to) = U4{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]),
                                            f32x2_to_bf16x2(v[4], v[5]), f32x2_to_bf16x2(v[6], v[7])};
        }
    }
    wave_lds_fence();
    T* out = static_cast<T*>(a.y) + n0 * a.ldy + kb * kBlockK;
    const int rows = (int)min((int64_t)kTileRows, a.N - n0), cols = min(kBlockK, a.K - kb * kBlockK);
    if constexpr (VEC) {
        constexpr int kRuns = kBlockK / kPer;      // 16-byte runs of a row
#pragma unroll
        for (int o = lane; o < kTileRows * kRuns; o += 64) {
            const int row = o / kRuns, k = o % kRuns * kPer;
            const T* from = &s_row[wave][row * kPitch + k];
            if (row >= rows) continue;
            if (k + kPer <= cols) {
                *reinterpret_cast<U4*>(out + row * a.ldy + k) = *reinterpret_cast<const U4*>(from);
            } else {
                for (int e = k; e < cols; ++e) out[row * a.ldy + e] = from[e - k];
            }
        }
    } else {
#pragma unroll 4
        for (int o = lane; o < kTileRows * kBlockK; o += 64) {
            const int row = o / kBlockK, k = o % kBlockK;
            if (row < rows && k < cols) out[row * a.ldy + k] = s_row[wave][row * kPitch + k];
        }
    }
}

// (T, S, G, Z) of a call
#define MTL_W4_G(KERNEL, T, S, Z, ...)                                             \
    switch (group) {                                                               \
        case 32: hipLaunchKernelGGL((KERNEL(T, S, 32, Z)), __VA_ARGS__); break;    \
        case 64: hipLaunchKernelGGL((KERNEL(T, S, 64, Z)), __VA_ARGS__); break;    \
        default: hipLaunchKernelGGL((KERNEL(T, S, 128, Z)), __VA_ARGS__); break;   \
    }
#define MTL_LINEAR_1(T, S, G, Z) linear_w4_kernel<T, S, G, Z, 1>
#define MTL_LINEAR_2(T, S, G, Z) linear_w4_kernel<T, S, G, Z, 2>
#define MTL_MATRIX(T, S, G, Z) dequantize_w4_kernel<T, S, G, Z, false>
#define MTL_MATRIX_VEC(T, S, G, Z) dequantize_w4_kernel<T, S, G, Z, true>
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
                   (int)((p->K + kBlockK - 1) / kBlockK), p->y_f32 != 0};
    const int parts = dtype == MTL_F32 ? 3 : 1;
    LinearW4 l{a, 0, 0, 1, 0};
    const int tiles = (a.N + kTileRows - 1) / kTileRows;
    // Rows of x to a workgroup: one operand tile's (16, of fp32 x 5) while that makes at most 2048 (tile of W, rows of x)
    // pairs, two tiles' where there are more: W is then read half as often.  Wavefronts to a pair: so many that the pairs
    // make about 2048; pairs to a workgroup: so many that it has 8 wavefronts.  Measured, GPU us (pairs; chosen, its
    // neighbours): 768x1536 1 row bf16 (48) 3.8, 4 / 2 wavefronts 4.2 / 4.5; 8192x2048 16 rows bf16 (512) 7.0, 8 / 2 8.8 /
    // 8.4; 8192x2048 8 rows fp32 (1024) 7.5, 4 / 1 8.7 / 9.7; 50280x2048 8 rows fp32 (6286) two tiles 19.4, one 27.3;
    // 2048x4096 64 rows bf16 (512) 9.8, two tiles 15.1.
    // A workgroup whose LDS has a CU to itself has 16 wavefronts, unless 8 make no more workgroups than CUs (16 would
    // leave CUs idle).  fp32, 16 / 8 wavefronts (workgroups of 8): 64 rows of 8192x2048 (448) 18.0 / 20.1, 12 of 20000x2048
    // (314) 17.8 / 19.1; 32 of 8192x2048 (256) 17.4 / 11.9, 48 of 2048x4096 (160) 24.7 / 16.8.
    const auto chunks_of = [&](int tm) { return (a.M + tm * 16 / parts - 1) / (tm * 16 / parts); };
    int tm = tiles * (int64_t)chunks_of(1) <= 2048 ? 1 : 2;
    const int chunks = chunks_of(tm);
    l.rows = (a.M + chunks - 1) / chunks;
    tm = (l.rows * parts + 15) / 16;
    const int pairs = (int)std::min<int64_t>(tiles * (int64_t)chunks, 1 << 20);
    const int per_block = kBlockK * 2 * parts * l.rows, pad = 16 * parts * l.rows;
    // (a block of x takes at most 8 KiB, so at least 8 fit)
    const auto blocks_of = [&](int waves) { return std::min(a.KB, (kLdsBytes - waves * tm * 1024 - pad) / per_block); };
    l.kblocks = blocks_of(8);
    while (l.wk < 8 && l.wk * 2 * pairs <= 2048 && l.wk * 2 <= a.KB) l.wk *= 2;
    int wn = std::min(8 / l.wk, std::max(2, pairs / 64));
    const bool two = (size_t)l.kblocks * per_block + pad + 8 * tm * 1024 <= kLdsBytes / 2;
    if (l.wk == 1 && !two && (int64_t)((tiles + 7) / 8) * chunks > 256) {
        wn = 16;
        l.kblocks = blocks_of(16);
    }
    if (l.kblocks < a.KB) {                                  // whole batches of every wavefront in each part of x
        while (l.wk > 1 && l.wk * kAhead > l.kblocks) l.wk /= 2, wn *= 2;
        l.kblocks -= l.kblocks % (l.wk * kAhead);
    }
    l.wk_log2 = __builtin_ctz(l.wk);
    const size_t lds = (size_t)l.kblocks * per_block + pad + wn * l.wk * tm * 1024;
    const int64_t groups = (tiles + wn - 1) / wn, most = two ? 512 : 256, passes = (groups * chunks + most - 1) / most;
    const dim3 grid((unsigned)((groups + passes - 1) / passes), chunks);
    switch (tm) {
        case 1: MTL_W4(MTL_LINEAR_1, grid, dim3(wn * l.wk * 64), lds, as_stream(stream), l) break;
        default: MTL_W4(MTL_LINEAR_2, grid, dim3(wn * l.wk * 64), lds, as_stream(stream), l) break;
    }
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
                   (int)((K + kBlockK - 1) / kBlockK), 0};
    const int64_t groups = ((N + kTileRows - 1) / kTileRows * a.KB + 3) / 4, gy = (groups + (1 << 22) - 1) >> 22;
    const dim3 grid((unsigned)((groups + gy - 1) / gy), (unsigned)gy);
    if (reinterpret_cast<uintptr_t>(W) % 16 == 0 && ldw * (dtype == MTL_F32 ? 4 : 2) % 16 == 0) {
        MTL_W4(MTL_MATRIX_VEC, grid, dim3(256), 0, as_stream(stream), a)
    } else {
        MTL_W4(MTL_MATRIX, grid, dim3(256), 0, as_stream(stream), a)
    }
    return check_launch("dequantize_w4");
}
