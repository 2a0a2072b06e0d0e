// The root-mean-square norm with the residual's addition, into eight bits and bf16: the entry, and the kernels for rows of bf16.
#include "q8_rows.cuh"

namespace t0 {
namespace q8 {

cudaError_t launch_norm_bf16(t0_runtime* rt, Rows& P) {
    return !P.residual ? launch_by_dim<true, false, kNone>(rt, P) : P.residual_f32 ? launch_by_dim<true, false, kF32>(rt, P) : launch_by_dim<true, false, kBf16>(rt, P);
}

}  // namespace q8
}  // namespace t0

using namespace t0;
using namespace t0::q8;

extern "C" {

int t0_q8_rmsnorm(t0_runtime* rt, const t0_q8_rmsnorm_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_rmsnorm_args a = *args;
    const uint32_t x_size = a.x_f32 ? 4 : 2, r_size = a.residual_f32 ? 4 : 2, w_size = a.weight_f32 ? 4 : 2;
    int rc = check_dim(a.n_rows, a.dim, kMaxRowDim);
    if (rc != T0_OK) return rc;
    if (!(a.eps >= 0.0f) || std::isinf(a.eps)) return fail(T0_ERR_INVALID, "eps=%g must be finite and not negative", (double)a.eps);
    if (a.n_rows == 0) return check_rt(rt);
    if (!a.x || !a.weight) return fail(T0_ERR_INVALID, "null device pointer");
    if (!a.q && !a.scales && !a.y) return fail(T0_ERR_INVALID, "null device pointer: neither rows in eight bits nor bf16 rows are asked for");
    if (!a.residual && a.residual_out) return fail(T0_ERR_INVALID, "residual_out without a residual");
    if (a.weight & 15) return fail(T0_ERR_INVALID, "the weight must be 16-byte aligned");
    if ((rc = kv4::check_rows("x", a.x, &a.x_stride, a.dim, x_size)) != T0_OK) return rc;
    if (a.residual && (rc = kv4::check_rows("residual", a.residual, &a.residual_stride, a.dim, r_size)) != T0_OK) return rc;
    if (a.residual_out && (rc = kv4::check_rows("residual_out", a.residual_out, &a.residual_out_stride, a.dim, r_size)) != T0_OK) return rc;
    if (a.y && (rc = kv4::check_rows("y", a.y, &a.y_stride, a.dim, 2)) != T0_OK) return rc;
    if ((a.q || a.scales) && (rc = check_codes("q", a.q, a.scales, &a.q_stride, a.dim)) != T0_OK) return rc;
    // what is read and what is written, in bytes
    struct Span { uint64_t at, bytes, step, rows; } in[3] = {{a.x, (uint64_t)a.dim * x_size, (uint64_t)a.x_stride * x_size, a.n_rows},
                                                             {a.residual, (uint64_t)a.dim * r_size, (uint64_t)a.residual_stride * r_size, a.n_rows},
                                                             {a.weight, (uint64_t)a.dim * w_size, (uint64_t)a.dim * w_size, 1}};
    const Span out[4] = {{a.residual_out, (uint64_t)a.dim * r_size, (uint64_t)a.residual_out_stride * r_size, a.n_rows},
                         {a.q, a.dim, a.q_stride, a.n_rows}, {a.scales, 4, 4, a.n_rows}, {a.y, (uint64_t)a.dim * 2, (uint64_t)a.y_stride * 2, a.n_rows}};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 3; ++i) {
            const bool itself = o == 0 && i < 2 && out[o].at == in[i].at && (i == 1 || x_size == r_size) && (out[o].step == in[i].step || a.n_rows == 1);
            if (!itself && touch(out[o].at, out[o].bytes, out[o].step, out[o].rows, in[i].at, in[i].bytes, in[i].step, in[i].rows))
                return fail(T0_ERR_INVALID, "what is written overlaps what is read (residual_out may be residual or x itself)");
        }
        for (int p = 0; p < o; ++p)
            if (touch(out[o].at, out[o].bytes, out[o].step, out[o].rows, out[p].at, out[p].bytes, out[p].step, out[p].rows))
                return fail(T0_ERR_INVALID, "arrays that are written overlap");
    }
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    Rows P;
    memset(&P, 0, sizeof P);
    P.x = (const void*)a.x; P.residual = (const void*)a.residual; P.weight = (const void*)a.weight; P.residual_out = (void*)a.residual_out;
    P.q = (int8_t*)a.q; P.scales = (float*)a.scales; P.y = (__nv_bfloat16*)a.y;
    P.x_stride = a.x_stride; P.residual_stride = a.residual_stride; P.residual_out_stride = a.residual_out_stride; P.q_stride = a.q_stride; P.y_stride = a.y_stride;
    P.n_rows = a.n_rows; P.dim = a.dim;
    P.inv_dim = 1.0 / a.dim; P.eps = a.eps;
    P.x_f32 = a.x_f32 != 0; P.residual_f32 = a.residual_f32 != 0; P.weight_f32 = a.weight_f32 != 0;
    prepare_rows(rt, P);
    const DeviceGuard guard(rt->device);
    return finish_rows(rt, P.x_f32 ? launch_norm_f32(rt, P) : launch_norm_bf16(rt, P));
}

}  // extern "C"
