// A decode step of a stack whose in_proj and out_proj are 4-bit matrices, in one C call (MambaLM.step at 1-32 rows,
// reference model.py:343-353 over MambaBlock.step 308-311 and MambaMixer.step 249-294).
//
// Launched op by op from Python a layer costs the host about 80 us (bf16, whose small parameters are then copied to
// fp32 each step, 140), which bounds an eager step; here it is six or seven launches:
//   in_proj from the codes (mtl_linear_w4) -> conv step + SiLU, the history shifted in place, with x_proj's partial sums
//   of each channel block (fp32: mtl_conv_step_xproj; bf16: the conv step, then x_proj as split-K parts on the matrix
//   cores) -> the partials summed in order -> the SSM update in place, y -> out_proj from the codes into floats -> the
//   residual add and the next RMSNorm.
// Captured steps at the mamba-1.4b width (48 layers, vocabulary 50280, groups of 128, the head in 4 bits too), against
// the same model's fp32 or bf16 weights: fp32 1 row 1388 -> 1114 us, 8 rows 1851 -> 1510, 32 rows 2318 -> 2195; bf16
// 1208 -> 1092, 1440 -> 1477, 1712 -> 1831.  At the mamba-130m width (24 layers) all are slower: fp32 321 -> 465, 539 ->
// 573, 616 -> 658; bf16 393 -> 442, 482 -> 576, 549 -> 623.  What is left beside the projections bounds it: six launches
// of about 4 us a layer, and matrix work that the wider weights' kernels fuse with the conv step.  Eager 1 row fp32 at
// the mamba-1.4b width: 3839 op by op, 1275 here.
#include <hip/hip_runtime.h>

#include <string>

#include "common.h"
#include "step_ops.h"

namespace {

using namespace mtl;

// split-K parts of the bf16 x_proj: whole 64-column runs, at least 4 to a part
int xproj_split(int32_t D) {
    int ks = 1;
    for (int p = 2; p <= 16; ++p)
        if (D % (64 * p) == 0 && D >= 256 * p) ks = p;
    return ks;
}

template <typename T>
int layers_w4(const mtl_decode_step_batched_args* a, const mtl_decode_layer* layers, const mtl_w4_matrix* mats,
              mtl_stream_t stream) {
    constexpr bool kF32 = sizeof(T) == 4;
    const int32_t b = a->batch, M = a->d_model, D = a->d_inner, N = a->d_state, R = a->dt_rank, K = a->d_conv;
    const int32_t J = R + 2 * N, nl = a->n_layers;
    auto t = [](const void* p) { return static_cast<const T*>(p); };
    auto w = [](void* p) { return static_cast<T*>(p); };
    T *inp = w(a->inp), *xc = w(a->xc), *xz = w(a->z), *y = w(a->y);
    auto linear = [&](const T* x, const mtl_w4_matrix& m, const void* bias, void* out, int64_t n, int64_t k, int f32) {
        const mtl_linear_w4_args l{x, m.codes, m.scales, m.zeros, bias, out, k, n, b, n, k, m.group,
                                   kF32 ? MTL_F32 : MTL_BF16, m.scale_dtype, f32};
        return mtl_linear_w4(&l, stream);
    };
    int rc = add_rmsnorm<T>(a->h, nullptr, 0, nullptr, t(layers[0].norm_w), inp, b, M, layers[0].eps, stream);
    if (rc) return rc;
    for (int32_t i = 0; i < nl; ++i) {
        const mtl_decode_layer& L = layers[i];
        const bool last = i + 1 == nl;
        if ((rc = linear(inp, mats[2 * i], L.b_in, xz, 2 * (int64_t)D, M, 0))) return rc;
        int parts;
        if constexpr (kF32) {
            parts = (D + 31) / 32;
            rc = mtl_conv_step_xproj(L.conv_state, xz, 2 * (int64_t)D, L.conv_w, L.conv_b, xc, D, L.W_xT, a->xpart, b,
                                     D, K, J, stream);
        } else {
            parts = xproj_split(D);
            rc = conv_step_bf16(w(L.conv_state), xz, 2 * (int64_t)D, t(L.conv_w), t(L.conv_b), xc, D, b, D, K, stream);
            if (rc) return rc;
            rc = linear_parts<T>(xc, D, t(L.W_x), nullptr, a->xpart, J, (int64_t)b * J, b, J, D, parts, 16, stream);
        }
        if (rc) return rc;
        if ((rc = mtl_sum_parts(a->xpart, parts, (int64_t)b * J, a->x_dbl, stream))) return rc;
        rc = state_update<T>(L.ssm_state, xc, D, xz + D, 2 * (int64_t)D, a->x_dbl, J, t(L.W_dt), t(L.dt_bias),
                             t(L.A_log), t(L.Dv), y, D, b, D, N, R, stream);
        if (rc) return rc;
        if ((rc = linear(y, mats[2 * i + 1], L.b_out, a->parts, M, D, 1))) return rc;
        rc = add_rmsnorm<T>(a->h, a->parts, 1, a->h, t(last ? a->norm_f : layers[i + 1].norm_w),
                            last ? w(a->normed_out) : inp, b, M, last ? a->eps_f : layers[i + 1].eps, stream);
        if (rc) return rc;
    }
    return MTL_OK;
}

}  // namespace

extern "C" int mtl_decode_step_w4(const mtl_decode_step_batched_args* a, const mtl_decode_layer* layers,
                                  const mtl_w4_matrix* matrices, int32_t dtype, mtl_stream_t stream) {
    clear_error();
    MTL_REQUIRE(a && layers && matrices, "null args, layers or matrices");
    MTL_REQUIRE(dtype == MTL_F32 || dtype == MTL_BF16, "dtype must be MTL_F32 or MTL_BF16");
    const bool bf16 = dtype == MTL_BF16;
    const int32_t b = a->batch, M = a->d_model, D = a->d_inner, N = a->d_state, R = a->dt_rank, K = a->d_conv;
    const int32_t J = R + 2 * N;
    MTL_REQUIRE(b >= 1 && b <= 32, "batch must be in [1, 32]");
    MTL_REQUIRE(a->n_layers >= 1, "n_layers must be >= 1");
    MTL_REQUIRE(M >= 1 && M <= 65536 && D >= 1 && D <= 65536, "d_model and d_inner must be in [1, 65536]");
    MTL_REQUIRE(N >= 1 && N <= 16 && R >= 1 && R <= 256 && J <= 288,
                "d_state must be in [1, 16], dt_rank in [1, 256], their J at most 288");
    MTL_REQUIRE(K >= 2 && K <= 4, "d_conv must be 2, 3 or 4");
    MTL_REQUIRE(!bf16 || (D % 64 == 0 && D >= 256 && J % 4 == 0),
                "bf16: d_inner must be a multiple of 64, at least 256, and dt_rank + 2 d_state of 4");
    MTL_REQUIRE(a->fold == 0, "there is no folded form");
    MTL_REQUIRE(a->h && a->inp && a->xc && a->z && a->y && a->xpart && a->x_dbl && a->parts && a->norm_f &&
                a->normed_out, "null workspace pointer");
    auto al16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    MTL_REQUIRE(al16(a->xc) && al16(a->xpart), "workspace xc and xpart must be 16-byte aligned");
    MTL_REQUIRE(a->inp != a->h && a->normed_out != a->h && a->normed_out != a->parts,
                "inp and normed_out must not alias h (normed_out not parts either)");
    // every layer before the first launch: a bad one leaves no conv history or SSM state half stepped
    for (int32_t i = 0; i < a->n_layers; ++i) {
        const mtl_decode_layer& L = layers[i];
        const std::string at = "layer " + std::to_string(i) + ": ";
        MTL_REQUIRE(L.norm_w && L.conv_w && (bf16 ? L.W_x : L.W_xT) && L.W_dt && L.dt_bias && L.A_log &&
                    L.conv_state && L.ssm_state, at + "null required pointer");
        MTL_REQUIRE(!bf16 || al16(L.W_x), at + "W_x must be 16-byte aligned");
        for (int j = 0; j < 2; ++j) {
            const mtl_w4_matrix& m = matrices[2 * i + j];
            MTL_REQUIRE(m.codes && m.scales && al16(m.codes) && al16(m.scales) &&
                        reinterpret_cast<uintptr_t>(m.zeros) % 4 == 0,
                        at + "codes and scales must be there and 16-byte aligned, zeros 4-byte aligned");
            MTL_REQUIRE(m.group == 32 || m.group == 64 || m.group == 128, at + "group must be 32, 64 or 128");
            MTL_REQUIRE(m.scale_dtype == MTL_F32 || m.scale_dtype == MTL_BF16,
                        at + "scale_dtype must be MTL_F32 or MTL_BF16");
        }
    }
    return bf16 ? layers_w4<uint16_t>(a, layers, matrices, stream) : layers_w4<float>(a, layers, matrices, stream);
}
