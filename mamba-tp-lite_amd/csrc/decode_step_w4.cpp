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

#include "decode_step_quant.h"

namespace {

using namespace mtl;

template <typename T>
int layers_w4(const mtl_decode_step_batched_args* a, const mtl_decode_layer* layers, const mtl_w4_matrix* mats,
              mtl_stream_t stream) {
    constexpr bool kF32 = sizeof(T) == 4;
    const int32_t b = a->batch, M = a->d_model, D = a->d_inner, nl = a->n_layers;
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
        if ((rc = step_between<T>(a, L, xz, xc, y, stream))) return rc;
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
    // every layer before the first launch: a bad one leaves no conv history or SSM state half stepped
    const std::string bad = check_quant_step(a, layers, dtype);
    MTL_REQUIRE(bad.empty(), bad);
    for (int32_t i = 0; i < a->n_layers; ++i) {
        const std::string at = "layer " + std::to_string(i) + ": ";
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
    return dtype == MTL_BF16 ? layers_w4<uint16_t>(a, layers, matrices, stream) : layers_w4<float>(a, layers, matrices, stream);
}
