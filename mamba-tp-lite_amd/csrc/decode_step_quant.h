// What the one-call decode steps of quantized stacks share (decode_step_w4.cpp, decode_step_int8.cpp): a layer between its
// in_proj and its out_proj, and the checks of everything but the projections' matrices.
#pragma once

#include <string>

#include "common.h"
#include "step_ops.h"

namespace mtl {

// split-K parts of the bf16 x_proj: whole 64-column runs, at least 4 to a part
inline int xproj_split(int32_t D) {
    int ks = 1;
    for (int p = 2; p <= 16; ++p)
        if (D % (64 * p) == 0 && D >= 256 * p) ks = p;
    return ks;
}

// xz [b, 2 D] -> y [b, D]: the conv step + SiLU, the history shifted in place, with x_proj's partial sums of each channel
// block (fp32: mtl_conv_step_xproj; bf16: the conv step, then x_proj as split-K parts on the matrix cores), the partials
// summed in order, and the SSM update in place.
template <typename T>
int step_between(const mtl_decode_step_batched_args* a, const mtl_decode_layer& L, const T* xz, T* xc, T* y,
                 mtl_stream_t stream) {
    const int32_t b = a->batch, D = a->d_inner, N = a->d_state, R = a->dt_rank, K = a->d_conv, J = R + 2 * N;
    auto t = [](const void* p) { return static_cast<const T*>(p); };
    auto w = [](void* p) { return static_cast<T*>(p); };
    int parts, rc;
    if constexpr (sizeof(T) == 4) {
        parts = (D + 31) / 32;
        rc = mtl_conv_step_xproj(L.conv_state, xz, 2 * (int64_t)D, L.conv_w, L.conv_b, xc, D, L.W_xT, a->xpart, b, D, K, J,
                                 stream);
    } else {
        parts = xproj_split(D);
        rc = conv_step_bf16(w(L.conv_state), xz, 2 * (int64_t)D, t(L.conv_w), t(L.conv_b), xc, D, b, D, K,
                            stream);
        if (rc) return rc;
        rc = linear_parts<T>(xc, D, t(L.W_x), nullptr, a->xpart, J, (int64_t)b * J, b, J, D, parts, 16, stream);
    }
    if (rc) return rc;
    if ((rc = mtl_sum_parts(a->xpart, parts, (int64_t)b * J, a->x_dbl, stream))) return rc;
    return state_update<T>(L.ssm_state, xc, D, xz + D, 2 * (int64_t)D, a->x_dbl, J, t(L.W_dt), t(L.dt_bias), t(L.A_log),
                           t(L.Dv), y, D, b, D, N, R, stream);
}

// The sizes, the workspace and every layer's pointers, for the entry point `who`; empty: sound.
inline std::string check_quant_step(const mtl_decode_step_batched_args* a, const mtl_decode_layer* layers, int32_t dtype) {
    if (dtype != MTL_F32 && dtype != MTL_BF16) return "dtype must be MTL_F32 or MTL_BF16";
    const bool bf16 = dtype == MTL_BF16;
    const int32_t b = a->batch, M = a->d_model, D = a->d_inner, N = a->d_state, R = a->dt_rank, K = a->d_conv;
    const int32_t J = R + 2 * N;
    if (!(b >= 1 && b <= 32)) return "batch must be in [1, 32]";
    if (!(a->n_layers >= 1)) return "n_layers must be >= 1";
    if (!(M >= 1 && M <= 65536 && D >= 1 && D <= 65536)) return "d_model and d_inner must be in [1, 65536]";
    if (!(N >= 1 && N <= 16 && R >= 1 && R <= 256 && J <= 288))
        return "d_state must be in [1, 16], dt_rank in [1, 256], their J at most 288";
    if (!(K >= 2 && K <= 4)) return "d_conv must be 2, 3 or 4";
    if (bf16 && !(D % 64 == 0 && D >= 256 && J % 4 == 0))
        return "bf16: d_inner must be a multiple of 64, at least 256, and dt_rank + 2 d_state of 4";
    if (a->fold != 0) return "there is no folded form";
    if (!(a->h && a->inp && a->xc && a->z && a->y && a->xpart && a->x_dbl && a->parts && a->norm_f && a->normed_out))
        return "null workspace pointer";
    if (!(al16(a->xc) && al16(a->xpart))) return "workspace xc and xpart must be 16-byte aligned";
    if (!(a->inp != a->h && a->normed_out != a->h && a->normed_out != a->parts))
        return "inp and normed_out must not alias h (normed_out not parts either)";
    for (int32_t i = 0; i < a->n_layers; ++i) {
        const mtl_decode_layer& L = layers[i];
        const std::string at = "layer " + std::to_string(i) + ": ";
        if (!(L.norm_w && L.conv_w && (bf16 ? L.W_x : L.W_xT) && L.W_dt && L.dt_bias && L.A_log && L.conv_state && L.ssm_state))
            return at + "null required pointer";
        if (bf16 && !al16(L.W_x)) return at + "W_x must be 16-byte aligned";
    }
    return "";
}

}  // namespace mtl
