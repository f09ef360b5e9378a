// A decode step of a stack whose in_proj and out_proj are matrices in 8-bit integers, in one C call (MambaLM.step at 1-32
// rows, reference model.py:343-353 over MambaBlock.step 308-311 and MambaMixer.step 249-294).
//
// Per layer seven or eight launches: in_proj in int8 (mtl_linear_int8) on the rows that the norm before it left -> the conv
// step, x_proj's parts and their sum, the SSM update (step_between) -> y in int8 (mtl_quantize_int8) -> out_proj into floats
// -> the residual add and the next RMSNorm in int8 (mtl_add_rmsnorm_int8), norm_f's in `dtype`.  At batch 1 the norm goes with
// its in_proj and the codes of y with out_proj (mtl_row_linear_int8): two launches fewer, and the same values.
#include <hip/hip_runtime.h>

#include <utility>

#include "decode_step_quant.h"
#include "int8.h"

namespace {

using namespace mtl;

template <typename T>
int layers_int8(const mtl_decode_step_batched_args* a, const mtl_decode_layer* layers, const mtl_int8_matrix* mats,
                mtl_stream_t stream) {
    constexpr int32_t kType = sizeof(T) == 4 ? MTL_F32 : MTL_BF16;
    const int32_t b = a->batch, M = a->d_model, D = a->d_inner, nl = a->n_layers;
    auto t = [](const void* p) { return static_cast<const T*>(p); };
    auto w = [](void* p) { return static_cast<T*>(p); };
    T *xc = w(a->xc), *xz = w(a->z), *y = w(a->y);
    int8_t *in = reinterpret_cast<int8_t*>(a->inp), *yq = reinterpret_cast<int8_t*>(a->xn);
    float *in_s = a->sq, *yq_s = a->sq + b;
    auto linear = [&](const int8_t* x, const float* s, const mtl_int8_matrix& m, const void* bias, void* out, int64_t n,
                      int64_t k, int32_t f32) {
        const mtl_linear_int8_args l{x, s, m.codes, m.scales, bias, out, n, b, n, k, kType, f32};
        return mtl_linear_int8(&l, stream);
    };
    auto norm = [&](const float* parts, const mtl_decode_layer& L) {
        const mtl_add_rmsnorm_int8_args n{a->h, parts, parts ? a->h : nullptr, L.norm_w, in, in_s, b, M, L.eps, MTL_F32,
                                          kType, 0};
        return mtl_add_rmsnorm_int8(&n, stream);
    };
    const bool row_in = b == 1 && row_linear_int8_pays(2 * (int64_t)D, M, true);
    const bool row_out = b == 1 && row_linear_int8_pays(M, D, false);
    // (every workgroup of an in_proj that norms reads h, so the sum goes to another buffer)
    float *h = a->h, *next = a->inp;
    int rc = row_in ? MTL_OK : norm(nullptr, layers[0]);
    for (int32_t i = 0; i < nl && !rc; ++i) {
        const mtl_decode_layer& L = layers[i];
        if (row_in) {
            const mtl_row_linear_int8_args r{h, i ? a->parts : nullptr, i ? next : nullptr, L.norm_w, mats[2 * i].codes,
                                             mats[2 * i].scales, L.b_in, xz, 2 * (int64_t)D, M, L.eps, kType, 0, 0};
            rc = mtl_row_linear_int8(&r, stream);
            if (i) std::swap(h, next);
        } else {
            rc = linear(in, in_s, mats[2 * i], L.b_in, xz, 2 * (int64_t)D, M, 0);
        }
        if (rc || (rc = step_between<T>(a, L, xz, xc, y, stream))) return rc;
        if (row_out) {
            const mtl_row_linear_int8_args r{y, nullptr, nullptr, nullptr, mats[2 * i + 1].codes, mats[2 * i + 1].scales,
                                             L.b_out, a->parts, M, D, 0.f, kType, 1, 0};
            rc = mtl_row_linear_int8(&r, stream);
        } else {
            if ((rc = mtl_quantize_int8(y, D, yq, yq_s, b, D, kType, stream))) return rc;
            rc = linear(yq, yq_s, mats[2 * i + 1], L.b_out, a->parts, M, D, 1);
        }
        if (rc) return rc;
        if (i + 1 == nl)
            rc = add_rmsnorm<T>(h, a->parts, 1, a->h, t(a->norm_f), w(a->normed_out), b, M, a->eps_f, stream);
        else if (!row_in)
            rc = norm(a->parts, layers[i + 1]);
    }
    return rc;
}

}  // namespace

extern "C" int mtl_decode_step_int8(const mtl_decode_step_batched_args* a, const mtl_decode_layer* layers,
                                    const mtl_int8_matrix* matrices, int32_t dtype, mtl_stream_t stream) {
    clear_error();
    MTL_REQUIRE(a && layers && matrices, "null args, layers or matrices");
    // every layer before the first launch: a bad one leaves no conv history or SSM state half stepped
    const std::string bad = check_quant_step(a, layers, dtype);
    MTL_REQUIRE(bad.empty(), bad);
    MTL_REQUIRE(a->xn && a->sq, "null workspace pointer");
    MTL_REQUIRE(al16(a->inp) && al16(a->xn), "workspace inp and xn must be 16-byte aligned");
    for (int32_t i = 0; i < 2 * a->n_layers; ++i)
        MTL_REQUIRE(matrices[i].codes && matrices[i].scales && al16(matrices[i].codes),
                    "layer " + std::to_string(i / 2) + ": codes and scales must be there, codes 16-byte aligned");
    return dtype == MTL_BF16 ? layers_int8<uint16_t>(a, layers, matrices, stream)
                             : layers_int8<float>(a, layers, matrices, stream);
}
