// Products of two matrices of 8-bit integers with a scale for each row (gfx950):
//   y[m, n] = bias[n] + sx[m] sw[n] sum_k cx[m, k] cw[n, k]
// The sum is exact (32-bit integers), so neither its order nor the tile that takes it shows in the result.

#include "int8.h"

namespace mtl {
namespace {

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

// the float of a sum, each factor rounded once
__device__ __forceinline__ float scaled(int acc, float sx, float sw, float bias) { return fmaf((float)acc * sx, sw, bias); }

// 16 bytes per lane from base + off to LDS, at to + 16 lane, asynchronously (vmcnt).  In assembly because the compiler
// waits for every copy by the builtin before the next read of LDS, whatever slot it reads: one stage of a product then
// took a whole round trip to memory (256 rows, 2048 x 4096: 21 us).
__device__ __forceinline__ void copy_kilobyte(const int8_t* base, uint32_t off, uint8_t* to) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) uint8_t* Lds;
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(Lds)to);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(at) : "m0");
#else
    (void)base; (void)off; (void)to;
#endif
}

// T: y.  A workgroup takes BN columns by BM rows of y, a wavefront WN x WM of them as 16 x 16 MFMA tiles with the
// rows of W as the first operand, so that a lane holds 4 neighbouring columns of y.
template <typename T, int BN, int BM, int WN, int WM, int ST, int OCC>
__global__ void __launch_bounds__(BN / WN * (BM / WM) * 64, OCC) linear_int8_kernel(const LinearArgs a) {
    constexpr int NWM = BM / WM, NW = BN / WN * NWM, NT = NW * 64;
    constexpr int TJ = WN / 16, TI = WM / 16, KB = kInt8Pad, KS = KB / 64;     // MFMA tiles of a wavefront; steps of a stage
    constexpr int SROWS = BN + BM, STAGE = SROWS * KB;
    constexpr int CR = 1024 / KB, NC = KB / 16, NI = SROWS / CR / NW;   // rows of a 1 KB copy, chunks of a row, copies per wavefront
    static_assert(SROWS % (CR * NW) == 0 && BN % CR == 0, "copies divide over the wavefronts");
    constexpr int kPer = 16 / (int)sizeof(T), kOut = 16 * (WN + kPer);  // a wavefront's 16 rows of y in LDS
    constexpr int kEnd = NW * kOut * (int)sizeof(T) + 8 * BN, kLds = ST * STAGE > kEnd ? ST * STAGE : kEnd;
    __shared__ __align__(1024) uint8_t ring[kLds];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave / NWM, wm = wave % NWM;

    int t = blockIdx.x;
    const int total = a.tm * a.tn;
    {
        const int per = total / 8, rem = total % 8, x = t % 8, i = t / 8;
        t = x * per + min(x, rem) + i;
    }
    constexpr int GM = 8;
    const int group = t / (GM * a.tn), g0 = group * GM, gm = min(GM, a.tm - g0);
    const int in_g = t - group * GM * a.tn;
    const int m0 = __builtin_amdgcn_readfirstlane((g0 + in_g % gm) * BM);
    const int n0 = __builtin_amdgcn_readfirstlane(in_g / gm * BN);

    // copy g of a stage: its rows CR g ..; lane l puts a 16-byte chunk of row CR g + l / NC at position l % NC.  Chunk c of
    // a row stands at position c ^ swizzle(row): the 16 rows of a fragment's chunk then lie in different banks.
    auto swizzle = [](int row) __attribute__((always_inline)) { return row >> 1 & 7; };
    const int8_t* const wt = a.w + (int64_t)n0 * a.Kp;
    const int8_t* const xt = a.x + (int64_t)m0 * a.Kp;
    uint32_t off[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int row = CR * (wave * NI + i) + lane / NC;
        const int rr = row < BN ? min(row, a.N - 1 - n0) : min(row - BN, a.M - 1 - m0);
        off[i] = (uint32_t)rr * (uint32_t)a.Kp + 16u * (lane % NC ^ swizzle(row));
    }
    auto issue1 = [&](int i, int slot, int s) __attribute__((always_inline)) {
        copy_kilobyte((CR * (wave * NI + i) < BN ? wt : xt) + (uint32_t)s * KB, off[i], ring + slot * STAGE + (wave * NI + i) * 1024);
    };

    I4 acc[TJ][TI];
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int i = 0; i < TI; ++i) acc[j][i] = I4{0, 0, 0, 0};

    const int r16 = lane & 15, g4 = lane >> 4;
    uint32_t o[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) o[k] = r16 * KB + 16 * ((4 * k + g4) ^ swizzle(r16));
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
    // s + ST into its slot issued, between its products
    auto body = [&](Frag& cur, Frag& nxt, int s, int k) __attribute__((always_inline)) {
        const bool end = k + 1 == KS;
        const int H = end ? MT / 2 : 0, left = MT - H, prev = slot;
        bool load = false;
#pragma unroll
        for (int q = 0; q < H; ++q) mma1(cur, q);
        __builtin_amdgcn_sched_barrier(0);
        if (end) {
            if (s + 1 < ns) {
                if (s + ST > ns)
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                else
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * NI) : "memory");
            }
            load = s + ST < ns;
            slot = slot + 1 == ST ? 0 : slot + 1;                        // (after the last stage: read, never used)
        }
#pragma unroll
        for (int q = 0; q < left; ++q) {
            mma1(cur, H + q);
            if (end && load && q < (left + 1) / 2) {
#pragma unroll
                for (int i = 2 * q * NI / left; i < min(2 * (q + 1) * NI / left, NI); ++i) issue1(i, prev, s + ST);
            }
#pragma unroll
            for (int r = min(q * NR / left, NR); r < min((q + 1) * NR / left, NR); ++r)
                read1(nxt, r, slot, end ? 0 : k + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
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
    for (int s = 0; s < ns; ++s) {
        body(f0, f1, s, 0);
        body(f1, f0, s, 1);
    }

    // D[j][i] of a tile: column lane % 16 (a row m of y), row 4 (lane / 16) + q in register q (a column n)
    lds_barrier();
    T* const out = reinterpret_cast<T*>(ring) + wave * kOut;
    float* const s_sw = reinterpret_cast<float*>(ring + NW * kOut * sizeof(T));
    float* const s_b = s_sw + BN;
    for (int n = threadIdx.x; n < BN; n += NT) {
        const int nc = min(n0 + n, a.N - 1);
        s_sw[n] = a.sw[nc];
        s_b[n] = a.bias ? load_param(a.bias, nc, a.bias_bf16) : 0.f;
    }
    lds_barrier();
    const int nw = n0 + wn * WN;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const int mt = m0 + wm * WM + 16 * i;
        const float sx = a.sx[min(mt + r16, a.M - 1)];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            const int c = 16 * j + 4 * g4;
            const F4v sw = ld4(s_sw + wn * WN + c), b = ld4(s_b + wn * WN + c);
            F4v v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = scaled(acc[j][i][e], sx, sw[e], b[e]);
            st4(out + r16 * (WN + kPer) + c, v);
        }
        wave_lds_fence();
        if (a.vec && nw + WN <= a.N) {
            constexpr int RPR = WN / kPer, RP = 64 / RPR;      // 16-byte runs of a row; rows of an instruction
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += RP) {
                const int r = r0 + lane / RPR, c = lane % RPR * kPer;
                if (RP > 16 && r >= 16) break;
                const I4 v = *reinterpret_cast<const I4*>(out + r * (WN + kPer) + c);
                if (mt + r < a.M) *reinterpret_cast<I4*>(static_cast<T*>(a.y) + (int64_t)(mt + r) * a.ldy + nw + c) = v;
            }
        } else {
            for (int e = lane; e < 16 * WN; e += 64) {
                const int r = e / WN, c = e % WN;
                if (mt + r < a.M && nw + c < a.N) static_cast<T*>(a.y)[(int64_t)(mt + r) * a.ldy + nw + c] = out[r * (WN + kPer) + c];
            }
        }
        wave_lds_fence();
    }
}

// Few rows of x, bound by the stream of W and by latency: nothing is shared.  NW wavefronts take 16 columns by 16 rows of y
// together, each a run of K, straight from memory to registers with 4 steps of 64 columns on their way, and add their sums.
// (32 columns or rows to a workgroup: 1x768x1536 3.0 us -> 4.0 and 3.3.  W loaded as nontemporal: 3.6, its lines come twice.)
template <typename T, int NW> __global__ void __launch_bounds__(NW * 64) stream_int8_kernel(const LinearArgs a) {
    constexpr int U = 4;
    __shared__ __align__(16) I4 s_acc[NW][64];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int8_t* w = a.w + (int64_t)min(n0 + r16, a.N - 1) * a.Kp + 16 * g4;
    const int8_t* x = a.x + (int64_t)min(m0 + r16, a.M - 1) * a.Kp + 16 * g4;
    const int steps = a.Kp / 64, per = (steps + NW - 1) / NW, s0 = wave * per, s1 = min(s0 + per, steps);
    I4 acc = {0, 0, 0, 0}, fw[U], fx[U];
    auto load = [&](int u, int s) __attribute__((always_inline)) {
        const int k = min(s, steps - 1) * 64;                   // (past the run: loaded, never used)
        fw[u] = *reinterpret_cast<const I4*>(w + k);
        fx[u] = *reinterpret_cast<const I4*>(x + k);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) load(u, s0 + u);
    for (int s = s0; s < s1; s += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u < s1) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], fx[u], acc, 0, 0, 0);
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

template <int BN, int BM, int WN, int WM, int ST, int OCC> int launch(LinearArgs a, bool f32, hipStream_t st) {
    const int64_t tm = (a.M + (int64_t)BM - 1) / BM, tn = (a.N + (int64_t)BN - 1) / BN;
    MTL_REQUIRE(tm * tn < (int64_t(1) << 31), "too many output tiles");
    a.tm = (int)tm;
    a.tn = (int)tn;
    const dim3 grid((unsigned)(tm * tn)), nt(BN / WN * (BM / WM) * 64);
    if (f32) hipLaunchKernelGGL((linear_int8_kernel<float, BN, BM, WN, WM, ST, OCC>), grid, nt, 0, st, a);
    else hipLaunchKernelGGL((linear_int8_kernel<uint16_t, BN, BM, WN, WM, ST, OCC>), grid, nt, 0, st, a);
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
    MTL_REQUIRE(p->M <= int64_t(1) << 30, "M must be in [0, 2^30]");
    MTL_REQUIRE(act_dtype(p->dtype), "dtype must be MTL_F32 or MTL_BF16");
    if (p->M == 0) return MTL_OK;
    MTL_REQUIRE(p->x && p->x_scales && p->w && p->w_scales && p->y, "null pointer");
    MTL_REQUIRE(al16(p->x) && al16(p->w), "codes must be 16-byte aligned");
    MTL_REQUIRE(p->ldy >= p->N, "rows of y must not overlap");
    const bool f32 = p->dtype == MTL_F32 || p->y_f32;
    LinearArgs a{p->x, p->x_scales, p->w, p->w_scales, p->bias, p->y, p->ldy, (int)p->M, (int)p->N, (int)int8_row(p->K),
                 0, 0, al16(p->y) && p->ldy * (f32 ? 4 : 2) % 16 == 0, p->dtype == MTL_BF16};
    const hipStream_t st = as_stream(stream);
    // Few rows: the stream.  us at rows x N x K, bf16: 1x768x1536 3.0, tiles of 32 4.2; 64x768x1536 3.7 / 4.3, 128x768x1536
    // 5.5 / 4.4; 1x8192x2048 5.3 / 5.6, 32x8192x2048 9.7 / 5.9.  Eight wavefronts on long rows: 1x2048x4096 4.8, four 5.1;
    // 16x1536x768 3.3, four 2.8.
    const int64_t pairs = ((a.N + 15) / 16) * (int64_t)((a.M + 15) / 16);
    if (pairs <= (a.M <= 16 ? 512 : 256))
        return a.Kp > 2048 ? launch_stream<8>(a, f32, st) : launch_stream<4>(a, f32, st);
    // Up to 64 rows of a wide W, bound by its stream: 16x50280x2048 21.0 (tiles of 64 24.6, of 32 22.1), 64 rows 23.8 (27.1,
    // 34.1)
    const auto tiles = [&](int bn, int bm) { return ((a.N + (int64_t)bn - 1) / bn) * ((a.M + (int64_t)bm - 1) / bm); };
    if (a.M <= 64 && tiles(128, 64) >= 192) return launch<128, 64, 32, 32, 3, 2>(a, f32, st);
    // Others by the time that a tile's rounds over the 256 CUs take, in units of one of 256 x 128 tiles (K 2048: 22.5 us);
    // the small tiles share a CU.  us with 256 x 256, 256 x 128, 128 x 128, 64 x 64, 32 x 32 (N x M):
    //   1024x8192x2048 31.9 22.5 27.7 32.3 53.5; 512x8192x2048 27.8 18.5 13.1 16.7 27.4; 4096x8192x2048 77.9 88.4 124.7 150
    //   227; 4096x2048x4096 51.6 37.1 43.4 53.5 93.8; 1024x2048x4096 48.9 30.0 19.6 15.7 26.2; 256x2048x4096 46.5 28.5 18.3
    //   11.4 9.8; 4096x768x1536 25.0 16.6 11.7 12.0 18.6; 512x768x1536 22.1 14.4 9.6 6.5 5.5
    const auto rounds = [&](int bn, int bm) { return (double)((tiles(bn, bm) + 255) / 256); };
    const double cost[5] = {1.72 * rounds(256, 256), 1.0 * rounds(256, 128), 0.58 * rounds(128, 128),
                            0.15 + 0.14 * rounds(64, 64), 0.12 + 0.07 * rounds(32, 32)};
    switch (std::min_element(cost, cost + 5) - cost) {
        case 0: return launch<256, 256, 128, 64, 2, 1>(a, f32, st);
        case 1: return launch<256, 128, 64, 64, 3, 1>(a, f32, st);
        case 2: return launch<128, 128, 64, 32, 4, 1>(a, f32, st);
        case 3: return launch<64, 64, 32, 32, 3, 3>(a, f32, st);
        default: return launch<32, 32, 16, 16, 5, 4>(a, f32, st);
    }
}
