// Products of two matrices of 8-bit integers with a scale for each row (gfx950):
//   y[m, n] = bias[n] + sx[m] sw[n] sum_k cx[m, k] cw[n, k]
// The sum is exact (32-bit integers), so neither its order nor the tile that takes it shows in the result.

#include "int8.h"

namespace mtl {
namespace {

typedef int I4u __attribute__((ext_vector_type(4), aligned(2)));

struct LinearArgs {
    const int8_t* x; const float* sx;      // [M, Kp], [M]
    const int8_t* w; const float* sw;      // [N, Kp], [N]
    const void* bias;                      // [N] or null
    void* y;
    int64_t ldy;
    int M, N, Kp;
    int tm, tn;                            // tiles along M and N
    bool vec;                              // 16-byte aligned rows of y
    bool bias_bf16;
};

// Copies to LDS, asynchronous (vmcnt): 16 or 4 bytes per lane from base + off to `to` + 16 or 4 lane.  In assembly because
// the compiler waits for every copy by the builtin before the next read of LDS, whatever slot it reads: one stage of a
// product then took a whole round trip to memory (256 rows, 2048 x 4096: 21 us in place of 12).
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    typedef __attribute__((address_space(3))) const uint8_t* Lds;
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(Lds)p);
}
#if defined(__HIP_DEVICE_COMPILE__)
#define MTL_COPY_TO_LDS(WIDTH, HINT, base, off, to)                                                                  \
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_" WIDTH " %0, %1" HINT ::"v"(off), "s"(base),      \
                 "s"(lds_address(to))                                                                                \
                 : "m0")
#else
#define MTL_COPY_TO_LDS(WIDTH, HINT, base, off, to) (void)(base), (void)(off), (void)(to)
#endif

// a pointer that is the same for the whole wavefront, in SGPRs
template <typename P> __device__ __forceinline__ const P* uniform(const P* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const P*>((uint64_t)hi << 32 | lo);
}

// T: y.  A workgroup takes BN columns by BM rows of y, a wavefront WN x WM of them as 16 x 16 MFMA tiles with the rows of W
// as the first operand, so that a lane holds 4 neighbouring columns of y.  K runs through a ring of ST stages of 128 columns
// in LDS.
//
// CHAIN: a workgroup takes one tile after the other and its copies never pause: while a tile's last stages are multiplied,
// the next one's first are on their way, and its first fragments are read before the tile is written.  The tiles' own starts
// and ends took 93 of the 526 us of 32768 x 8192 x 2048.  Three stages of K at least: the next tile's scales go where the
// last one's were, and a barrier has to stand between.
//
// ONCE: no other workgroup reads these rows of W, which go past the caches (16 x 50280 x 2048 21.2 -> 18.7 us).  PAST: y does.
template <typename T, int BN, int BM, int WN, int WM, int ST, int OCC, bool CHAIN, bool ONCE, bool PAST>
__global__ void __launch_bounds__(BN / WN * (BM / WM) * 64, OCC) linear_int8_kernel(const LinearArgs a) {
    constexpr int NWM = BM / WM, NW = BN / WN * NWM, NT = NW * 64;
    constexpr int TJ = WN / 16, TI = WM / 16, KB = kInt8Pad, KS = 2;      // MFMA tiles of a wavefront; steps of a stage
    constexpr int SROWS = BN + BM, STAGE = SROWS * KB, NI = SROWS / 8 / NW;         // 1 KB copies per wavefront and stage
    static_assert(SROWS % (8 * NW) == 0 && BN % 8 == 0, "copies divide over the wavefronts");
    static_assert(!CHAIN || (ST == 2 && NT == BN + BM && NT % 64 == 0), "a chain's scales are a copy per wavefront");
    // a wavefront's 16 rows of y on their way out, OW columns at a time; the scales of the tile's columns and rows
    constexpr int kPer = 16 / (int)sizeof(T), OW = CHAIN ? 128 / (int)sizeof(T) : WN, kOut = 16 * (OW + kPer);
    constexpr int kRing = ST * STAGE, kEnd = NW * kOut * (int)sizeof(T) + (CHAIN ? 8 : 4) * SROWS + 4 * BN;
    constexpr int kLds = CHAIN ? kRing + kEnd : kRing > kEnd ? kRing : kEnd;
    __shared__ __align__(1024) uint8_t ring[kLds];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave / NWM, wm = wave % NWM;
    T* const out = reinterpret_cast<T*>(ring + (CHAIN ? kRing : 0)) + wave * kOut;
    float* s_sw = reinterpret_cast<float*>(ring + (CHAIN ? kRing : 0) + NW * kOut * sizeof(T));    // [BN], then [BM]
    float* s_next = s_sw + SROWS;                              // (a chain's next tile's)
    float* const s_b = s_sw + (CHAIN ? 2 : 1) * SROWS;         // [BN]

    // XCD-aware tile order (workgroups are dealt to the 8 XCDs round robin): each XCD takes a contiguous range of tiles,
    // ordered 8 row tiles by all column tiles, rows fastest, so the tiles resident on an XCD at one time share their operand
    // rows in its L2
    const int total = a.tm * a.tn, xcd = blockIdx.x % 8, per = total / 8, rem = total % 8;
    const int first = xcd * per + min(xcd, rem), count = per + (xcd < rem), stride = (gridDim.x + 7 - xcd) / 8;
    auto place = [&](int j, int& m, int& n) __attribute__((always_inline)) {
        constexpr int GM = 8;
        const int t = first + j, group = t / (GM * a.tn), g0 = group * GM, gm = min(GM, a.tm - g0);
        const int in_g = t - group * GM * a.tn;
        // (uniform, but the divisions run on the VALU: back to SGPRs)
        m = __builtin_amdgcn_readfirstlane((g0 + in_g % gm) * BM);
        n = __builtin_amdgcn_readfirstlane(in_g / gm * BN);
    };

    // copy g of a stage: its rows 8 g ..; lane l puts a 16-byte chunk of row 8 g + l / 8 at position l % 8.  Chunk c of a row
    // stands at position c ^ (row / 2 % 8): the 16 rows of a fragment's chunk then lie in different banks (counted: no
    // conflicts; with row % 8 half of the LDS cycles were).
    const int8_t *wt, *xt;
    int wlast, xlast;                                          // the tile's last rows of W and x that are there
    const int row8 = lane >> 3, chunk = 16 * ((lane & 7) ^ (lane >> 4));
    auto aim = [&](int m, int n) __attribute__((always_inline)) {
        wt = uniform(a.w + (int64_t)n * a.Kp);
        xt = uniform(a.x + (int64_t)m * a.Kp);
        wlast = a.N - 1 - n;
        xlast = a.M - 1 - m;
    };
    auto issue1 = [&](int i, int slot, int s) __attribute__((always_inline)) {
        const int g = wave * NI + i;
        const bool isw = 8 * g < BN;
        const int8_t* base = (isw ? wt : xt) + (uint32_t)s * KB;
        const int row = min(row8 + 8 * g - (isw ? 0 : BN), isw ? wlast : xlast);
        const uint32_t off = __umul24(row, a.Kp) + (chunk ^ (g & 1) << 6);        // (256 rows, Kp <= 2^17)
        if (ONCE && isw) MTL_COPY_TO_LDS("dwordx4", " nt", base, off, ring + slot * STAGE + g * 1024);
        else MTL_COPY_TO_LDS("dwordx4", "", base, off, ring + slot * STAGE + g * 1024);
    };
    // the tile's scales, 64 to a wavefront
    auto issue_scales = [&](int m, int n, float* to) __attribute__((always_inline)) {
        const bool col = wave * 64 < BN;
        const int at = threadIdx.x - (col ? 0 : BN);
        const float* base = uniform(col ? a.sw + n : a.sx + m);
        const uint32_t off = 4u * (uint32_t)min(at, col ? a.N - 1 - n : a.M - 1 - m);
        MTL_COPY_TO_LDS("dword", "", base, off, to + wave * 64);
    };

    I4 acc[TJ][TI];
    const int r16 = lane & 15, g4 = lane >> 4;
    uint32_t o[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) o[k] = r16 * KB + 16 * ((4 * k + g4) ^ (r16 >> 1));
    struct Frag { I4 w[TJ], x[TI]; };
    constexpr int NR = TI + TJ, MT = TI * TJ;
    auto read1 = [&](Frag& f, int r, int slot, int k) __attribute__((always_inline)) {
        const uint8_t* p = ring + slot * STAGE + o[k];
        if (r < TJ) f.w[r] = *reinterpret_cast<const I4*>(p + (wn * WN + 16 * r) * KB);
        else f.x[r - TJ] = *reinterpret_cast<const I4*>(p + (BN + wm * WM + 16 * (r - TJ)) * KB);
    };
    auto mma1 = [&](const Frag& f, int q) __attribute__((always_inline)) {
        const int j = q % TJ, i = q / TJ;
        acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[j], f.x[i], acc[j][i], 0, 0, 0);
    };

    const int ns = a.Kp / KB;
    int slot = 0;
    // step k of stage s (its fragments in cur): the next step's fragments are read, and at a stage's end the copies of stage
    // s + ST into its slot issued, between its products.  `more`: stages past the last are the next tile's.
    auto body = [&](Frag& cur, Frag& nxt, int s, int k, bool more) __attribute__((always_inline)) {
        const bool end = k + 1 == KS;
        const int H = end ? MT / 2 : 0, left = MT - H, prev = slot;
        bool load = false;
#pragma unroll
        for (int q = 0; q < H; ++q) mma1(cur, q);
        __builtin_amdgcn_sched_barrier(0);
        if (end) {
            if (CHAIN || s + 1 < ns) {
                if (CHAIN || s + ST > ns)
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                else
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * NI) : "memory");
            }
            load = s + ST < ns || more;
            slot = slot + 1 == ST ? 0 : slot + 1;                        // (after the last stage: read, never used)
        }
        const int ahead = CHAIN && s + ST >= ns ? s + ST - ns : s + ST;
#pragma unroll
        for (int q = 0; q < left; ++q) {
            mma1(cur, H + q);
            if (end && load && q < (left + 1) / 2) {
#pragma unroll
                for (int i = 2 * q * NI / left; i < min(2 * (q + 1) * NI / left, NI); ++i) issue1(i, prev, ahead);
            }
#pragma unroll
            for (int r = min(q * NR / left, NR); r < min((q + 1) * NR / left, NR); ++r)
                read1(nxt, r, slot, end ? 0 : k + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    int tile = blockIdx.x / 8, m0, n0, m1 = 0, n1 = 0;
    place(tile, m0, n0);
    aim(m0, n0);
    if constexpr (CHAIN) {
        issue_scales(m0, n0, s_sw);
        if (threadIdx.x < BN) s_b[threadIdx.x] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < ST; ++s)
        if (s < ns) {
#pragma unroll
            for (int i = 0; i < NI; ++i) issue1(i, s, s);
        }
    if (ns >= ST)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 1) * NI) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    Frag f0, f1;
#pragma unroll
    for (int r = 0; r < NR; ++r) read1(f0, r, 0, 0);

    for (;;) {
        const bool more = CHAIN && tile + stride < count;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int i = 0; i < TI; ++i) acc[j][i] = I4{0, 0, 0, 0};
        for (int s = 0; s < ns; ++s) {
            if constexpr (CHAIN) {
                if (more && s + ST == ns) {
                    place(tile + stride, m1, n1);
                    aim(m1, n1);
                    issue_scales(m1, n1, s_next);
                }
            }
            body(f0, f1, s, 0, more);
            body(f1, f0, s, 1, more);
        }

        // D[j][i] of a tile: column lane % 16 (a row m of y), row 4 (lane / 16) + q in register q (a column n)
        if constexpr (!CHAIN) lds_barrier();
        if (!CHAIN || a.bias) {
            for (int e = threadIdx.x; e < SROWS; e += NT) {
                if constexpr (!CHAIN) s_sw[e] = e < BN ? a.sw[min(n0 + e, a.N - 1)] : a.sx[min(m0 + e - BN, a.M - 1)];
                if (e < BN) s_b[e] = a.bias ? load_param(a.bias, min(n0 + e, a.N - 1), a.bias_bf16) : 0.f;
            }
            lds_barrier();
        }
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            const int mt = m0 + wm * WM + 16 * i;
            const float sx = s_sw[BN + wm * WM + 16 * i + r16];
#pragma unroll
            for (int j0 = 0; j0 < TJ; j0 += OW / 16) {
                const int nw = n0 + wn * WN + 16 * j0;
#pragma unroll
                for (int j = 0; j < OW / 16; ++j) {
                    const int c = 16 * j + 4 * g4;
                    // (the bias in LDS too: a load that may stand between the stores would wait for them)
                    const F4v sw = ld4(s_sw + wn * WN + 16 * j0 + c), b = ld4(s_b + wn * WN + 16 * j0 + c);
                    F4v v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = scaled(acc[j0 + j][i][e], sx, sw[e], b[e]);
                    st4(out + r16 * (OW + kPer) + c, v);
                }
                wave_lds_fence();
                constexpr int RPR = OW / kPer, RP = 64 / RPR;          // 16-byte runs of a row; rows of an instruction
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += RP) {
                    const int r = r0 + lane / RPR, c = lane % RPR * kPer;
                    if (RP > 16 && r >= 16) break;
                    const T* from = out + r * (OW + kPer) + c;
                    T* y = static_cast<T*>(a.y) + (int64_t)(mt + r) * a.ldy + nw + c;
                    const int n = mt + r < a.M ? a.N - nw - c : 0;     // columns of the run that are there
                    if (n >= kPer) {
                        const I4 v = *reinterpret_cast<const I4*>(from);
                        if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<I4*>(y));
                        else *reinterpret_cast<I4u*>(y) = v;           // (at any alignment of a row)
                    } else {
                        for (int e = 0; e < n; ++e) y[e] = from[e];
                    }
                }
                wave_lds_fence();
            }
        }
        if (!more) break;
        tile += stride;
        m0 = m1;
        n0 = n1;
        float* const done = s_sw;
        s_sw = s_next;
        s_next = done;
    }
}

// Few rows of x, bound by the stream of W and by latency: nothing is shared.  NW wavefronts take 16 columns by 16 rows of y
// together, each a run of K, straight from memory to registers with 2 steps of 128 columns on their way, and add their sums.
// A lane takes 32 bytes of its row in a step (the order of K is free where both operands have the same): whole 128-byte
// lines of 16 rows.  us, 16 bytes at a time with 4 steps of 64 columns: 16x8192x2048 7.2 -> 6.6, 64x768x1536 4.1 -> 3.6.
// (32 columns or rows to a workgroup: 1x768x1536 3.0 -> 4.0 and 3.3.  W past the caches 3.2: its lines are read twice.)
template <typename T, int NW> __global__ void __launch_bounds__(NW * 64) stream_int8_kernel(const LinearArgs a) {
    constexpr int U = 2;
    __shared__ __align__(16) I4 s_acc[NW][64];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int8_t* w = a.w + (int64_t)min(n0 + r16, a.N - 1) * a.Kp + 32 * g4;
    const int8_t* x = a.x + (int64_t)min(m0 + r16, a.M - 1) * a.Kp + 32 * g4;
    const int steps = a.Kp / 128, per = (steps + NW - 1) / NW, s0 = wave * per, s1 = min(s0 + per, steps);
    I4 acc = {0, 0, 0, 0}, fw[U][2], fx[U][2];
    auto load = [&](int u, int s) __attribute__((always_inline)) {
        const int k = min(s, steps - 1) * 128;                  // (past the run: loaded, never used)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            fw[u][h] = *reinterpret_cast<const I4*>(w + k + 16 * h);
            fx[u][h] = *reinterpret_cast<const I4*>(x + k + 16 * h);
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(u, s0 + u);
    for (int s = s0; s < s1; s += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u < s1) {
#pragma unroll
                for (int h = 0; h < 2; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u][h], fx[u][h], acc, 0, 0, 0);
            }
            if (s + U < s1) load(u, s + U + u);
        }
    }
    s_acc[wave][lane] = acc;
    lds_barrier();
    const int m = m0 + r16, n = n0 + 4 * g4;
    if (wave || m >= a.M) return;
#pragma unroll
    for (int v = 1; v < NW; ++v) acc += s_acc[v][lane];
    const float sx = a.sx[m];
    T* y = static_cast<T*>(a.y) + (int64_t)m * a.ldy + n;
    F4v v;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int nc = min(n + q, a.N - 1);
        v[q] = scaled(acc[q], sx, a.sw[nc], a.bias ? load_param(a.bias, nc, a.bias_bf16) : 0.f);
    }
    if (a.vec && n + 4 <= a.N) {
        st4(y, v);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (n + q < a.N) Act<T>::store(y + q, v[q]);
    }
}

template <int NW> int launch_stream(const LinearArgs& a, bool f32, hipStream_t st) {
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 15) / 16)), nt(NW * 64);
    if (f32) hipLaunchKernelGGL((stream_int8_kernel<float, NW>), grid, nt, 0, st, a);
    else hipLaunchKernelGGL((stream_int8_kernel<uint16_t, NW>), grid, nt, 0, st, a);
    return check_launch("linear_int8");
}

template <int BN, int BM, int WN, int WM, int ST, int OCC, bool CHAIN = false, bool ONCE = false, bool PAST = false>
int launch(LinearArgs a, bool f32, hipStream_t st) {
    const int64_t tm = (a.M + (int64_t)BM - 1) / BM, tn = (a.N + (int64_t)BN - 1) / BN;
    MTL_REQUIRE(tm * tn < (int64_t(1) << 31), "too many output tiles");
    a.tm = (int)tm;
    a.tn = (int)tn;
    const dim3 grid((unsigned)(CHAIN ? std::min<int64_t>(tm * tn, 256) : tm * tn)), nt(BN / WN * (BM / WM) * 64);
    if (f32) hipLaunchKernelGGL((linear_int8_kernel<float, BN, BM, WN, WM, ST, OCC, CHAIN, ONCE, PAST>), grid, nt, 0, st, a);
    else hipLaunchKernelGGL((linear_int8_kernel<uint16_t, BN, BM, WN, WM, ST, OCC, CHAIN, ONCE, PAST>), grid, nt, 0, st, a);
    return check_launch("linear_int8");
}

}  // namespace
}  // namespace mtl

extern "C" int mtl_linear_int8(const mtl_linear_int8_args* p, mtl_stream_t stream) {
    using namespace mtl;
    clear_error();
    MTL_REQUIRE(p, "null pointer");
    MTL_INT8_SIZES(p->M, p->K);
    MTL_REQUIRE(p->N >= 1 && p->N <= int64_t(1) << 27, "N must be in [1, 2^27]");
    MTL_REQUIRE(act_dtype(p->dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (p->M == 0) return MTL_OK;
    MTL_REQUIRE(p->x && p->x_scales && p->w && p->w_scales && p->y, "null pointer");
    MTL_REQUIRE(al16(p->x) && al16(p->w), "codes must be 16-byte aligned");
    MTL_REQUIRE(p->ldy >= p->N, "rows of y must not overlap");
    const bool f32 = p->dtype == MTL_F32 || p->y_f32;
    constexpr int64_t kMost = int64_t(1) << 29;                // rows whose tiles, of any size, are whole in 32 bits
    if (p->M > kMost) {
        mtl_linear_int8_args c = *p;
        for (int64_t m = 0; m < p->M; m += kMost) {
            c.x = p->x + m * int8_row(p->K);
            c.x_scales = p->x_scales + m;
            c.y = static_cast<uint8_t*>(p->y) + m * p->ldy * (f32 ? 4 : 2);
            c.M = std::min(kMost, p->M - m);
            if (const int rc = mtl_linear_int8(&c, stream)) return rc;
        }
        return MTL_OK;
    }
    LinearArgs a{p->x, p->x_scales, p->w, p->w_scales, p->bias, p->y, p->ldy, (int)p->M, (int)p->N, (int)int8_row(p->K),
                 0, 0, al16(p->y) && p->ldy * (f32 ? 4 : 2) % 16 == 0, p->dtype == MTL_BF16};
    const hipStream_t st = as_stream(stream);
    // Few rows: the stream.  us at rows x N x K, bf16, W from HBM: 1x768x1536 3.0, tiles of 32 4.5; 64x768x1536 3.6 / 4.6;
    // 1x8192x2048 5.4 / 6.3, 16x8192x2048 6.7 / 6.6, 16x2048x4096 6.4 / 8.9; 4x16384x2048
    // 8.1 / 8.2, 16 rows of it 10.2 / 8.4; 128x768x1536 5.5 / 4.4, 32x8192x2048 9.7 / 5.9.
    // Eight wavefronts from 1536 columns on: 1x768x1536 3.4 with four; 1x1536x768 2.9, with eight 3.0; 33x1001x777 3.4 / 3.9.
    const int64_t pairs = ((a.N + 15) / 16) * (int64_t)((a.M + 15) / 16);
    if (pairs <= (a.M <= 4 ? 1024 : a.M <= 16 ? 512 : 256))
        return a.Kp >= 1536 ? launch_stream<8>(a, f32, st) : launch_stream<4>(a, f32, st);
    // Up to 64 rows of a wide W, bound by its stream, in one tile of rows: 16x50280x2048 18.7 (128 x 64 19.2, 64 x 64 23.4, 32 x
    // 32 19.6), 64 rows 22.0 (64 x 64 26.0, 32 x 32 34.7); 16x24000x1024 6.9 (7.6 with the rule below), 16x8192x2048 9.5 (6.7).
    const auto tiles = [&](int bn, int bm) { return ((a.N + (int64_t)bn - 1) / bn) * ((a.M + (int64_t)bm - 1) / bm); };
    if (a.M <= 64 && tiles(128, 64) >= 160)
        return a.M <= 32 ? launch<128, 32, 32, 32, 4, 2, false, true>(a, f32, st)
                         : launch<128, 64, 32, 32, 3, 2, false, true>(a, f32, st);
    // Whole lines of y go past the L2s (32 MB) where those would hold them, since what they hold is written back when the kernel
    // ends, and where not even the MALL (256 MB) does.  us of the product / of it with the quantize_int8 that reads y next, kept
    // and past, at 280 sizes, over one y and over two in turn: fp32 512x8192x2048 (16 MB) 16.1 and 14.8 / 21.9 and 21.0, bf16
    // 16384x768x1536 (24 MB) 27.6 and 25.8 / 38.3 and 37.5.  At 28 MB the product gains 4% and the two lose 1% on average, at 30 MB 2%
    // and 2% (fp32 5120x1536x768 12.2 and 11.9 / 19.9 and 20.8); fp32 2048x8192x2048 (64 MB) 37.8 and 39.8 / 51.6 and 55.1.  At 256 MB
    // three of ten sizes lose 6%, at 320 one 5% (fp32 10240x8192x2048 173 and 182 / 245 and 253), from 384 on the two none (12288 rows of
    // it 212 and 218 / 309 and 303, bf16 32768x8192x2048 519 and 503 / 676 and 651, fp32 87381x1536x768 197 and 151 / 320 and 289).
    // Rows that end inside a line lose at any size (8184x50277x768 690 and 855).
    const int64_t row = p->ldy * (f32 ? 4 : 2), y_bytes = p->M * row;
    const bool lines = row % 128 == 0 && reinterpret_cast<uintptr_t>(p->y) % 128 == 0;
    const bool past = lines && y_bytes <= 28 << 20, large = lines && y_bytes >= 384 << 20;
    // Others by the time that their tiles take on the 256 CUs, in us: each round of a tile per CU has its start and end (longer
    // where rows of y end inside a line, or are floats) and its stages of K; two or more tiles share a CU, and a round of them
    // has the traffic of all.  Measured at 210 sizes of up to 32768 rows with every tile, the choice takes 1% more than the best of
    // them on average (a cost by rounds alone 7% more), 5-20% more at ten of them, most of those with one to three stages of K:
    // 80x19686x76 5.5 by the last one for 4.6, 692x5440x384 7.8 for 6.6, fp32 5694x478x170 7.3 for 6.3.  us with the tiles in the
    // table's order:
    //   bf16 1024x8192x2048 - 21 27 34 - 23; fp32 8192x768x1536 - 19.6 25.7 25.0 - 18.8; 1179x2304x4480 56 34 23 28 40 32;
    //   720x1167x3393 54 31 20 14 16 28; fp32 657x576x1280 24 14 9.6 6.1 5.2 11; fp32 14280x1685x1184 - - - - - 49 (60 of the
    //   first); 32768x8192x2048 496 by the first, 586 by the second
    constexpr struct { int bn, bm, share; double start, round, stage, inside, floats, traffic; } kTiles[6] = {
        {256, 256, 1, 0.00, 3.81, 1.26, 0.81, 3.90, 0.0}, {256, 128, 1, 0.34, 5.63, 0.80, 0.61, 1.39, 0.0},
        {128, 128, 1, 1.06, 3.09, 0.54, 0.45, 0.90, 0.0}, {64, 64, 3, 2.49, 0.54, 0.11, 0.06, 0.26, 0.26},
        {32, 32, 4, 2.22, 0.35, 0.06, 0.02, 0.02, 0.14},  {128, 128, 2, 1.47, 1.72, 0.08, 0.10, 0.75, 0.78}};
    const int stages = a.Kp / kInt8Pad;
    int best = 0;
    double least = 0;
    for (int i = stages > 2 ? 0 : 1; i < 6; ++i) {
        const auto& t = kTiles[i];
        const int64_t count = tiles(t.bn, t.bm);
        if (i > 0 && count >= 1 << 23) continue;               // (512 threads each at most, and a launch has fewer than 2^32)
        const int64_t rounds = (count + 255) / 256, full = (count + 256 * t.share - 1) / (256 * t.share);
        const double us = t.start + rounds * (t.round + t.stage * stages + (lines ? 0 : t.inside) + (f32 ? t.floats : 0)) +
                          full * t.traffic * stages;
        if (least == 0 || us < least) { least = us; best = i; }
    }
    MTL_REQUIRE(least > 0, "too many output tiles");
#define MTL_TILE(...) (past ? launch<__VA_ARGS__, false, false, true>(a, f32, st) : launch<__VA_ARGS__>(a, f32, st))
    switch (best) {
        case 0: return large ? launch<256, 256, 128, 64, 2, 1, true, false, true>(a, f32, st)
                             : launch<256, 256, 128, 64, 2, 1, true>(a, f32, st);
        case 1: return MTL_TILE(256, 128, 64, 64, 3, 1);
        case 2: return MTL_TILE(128, 128, 64, 32, 4, 1);
        case 3: return MTL_TILE(64, 64, 32, 32, 3, 3);
        case 4: return MTL_TILE(32, 32, 16, 16, 5, 4);
        default: return MTL_TILE(128, 128, 32, 64, 2, 2);
    }
#undef MTL_TILE
}
