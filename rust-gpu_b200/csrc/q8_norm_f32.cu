// The root-mean-square norm of rows of f32 (a translation unit of its own: the kernels of one type take long to compile).
#include "q8_rows.cuh"

namespace t0 {
namespace q8 {

cudaError_t launch_norm_f32(t0_runtime* rt, Rows& P) {
    return !P.residual ? launch_by_dim<true, true, kNone>(rt, P) : P.residual_f32 ? launch_by_dim<true, true, kF32>(rt, P) : launch_by_dim<true, true, kBf16>(rt, P);
}

}  // namespace q8
}  // namespace t0
