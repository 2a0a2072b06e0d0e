// Products of rows in eight bits with weights in eight bits: the entries, and a kernel that takes every shape.
#include "gemm_common.cuh"
#include "q8.cuh"
#include "runtime_internal.h"

namespace t0 {
namespace q8 {
namespace {

constexpr uint32_t kTile = 64, kStep = 64;

// Four codes of a row from `e` on, as a word; those from k on are zero.
__device__ __forceinline__ uint32_t word_at(const int8_t* row, uint32_t e, uint32_t k) {
    if (e >= k) return 0;
    const uint32_t w = *(const uint32_t*)(row + e);            // strides are multiples of 16: the word is the row's
    return k - e >= 4 ? w : w & ((1u << (8 * (k - e))) - 1);
}

// 64 x 64 numbers a block, 16 a thread.
template <bool kGated>
__global__ void __launch_bounds__(256) q8_gemm_kernel(const Product P) {
    constexpr int kW = kGated ? 2 : 1;
    __shared__ uint32_t as[kTile][kStep / 4 + 1], ws[kW][kTile][kStep / 4 + 1];
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint64_t tiles_n = (P.n + kTile - 1) / kTile;
    const uint64_t m0 = blockIdx.x / tiles_n * kTile, n0 = blockIdx.x % tiles_n * kTile;
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int32_t sum[kW][4][4] = {};
    for (uint32_t k0 = 0; k0 < P.k; k0 += kStep) {
        for (uint32_t i = threadIdx.x; i < kTile * kStep / 4; i += 256) {
            const uint32_t r = i / (kStep / 4), c = i % (kStep / 4);
            as[r][c] = m0 + r < P.m ? word_at(P.a + (m0 + r) * P.a_stride, k0 + 4 * c, P.k) : 0;
#pragma unroll
            for (int h = 0; h < kW; ++h) ws[h][r][c] = n0 + r < P.n ? word_at(P.w[h] + (n0 + r) * P.w_stride, k0 + 4 * c, P.k) : 0;
        }
        __syncthreads();
        for (uint32_t c = 0; c < kStep / 4; ++c)
#pragma unroll
            for (int h = 0; h < kW; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[h][i][j] = __dp4a((int)as[ty + 16 * i][c], (int)ws[h][tx + 16 * j][c], sum[h][i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
            if (r >= P.m || c >= P.n) continue;
            float v = scaled(sum[0][i][j], P.a_scales[r], P.w_scales[0][c]);
            if constexpr (kGated) v = __fmul_rn(activate(v, P.act), scaled(sum[kW - 1][i][j], P.a_scales[r], P.w_scales[1][c]));
            else if (P.bias) v = __fadd_rn(v, P.bias[c]);
            if (P.out_bf16) ((__nv_bfloat16*)P.y)[r * P.y_stride + c] = __float2bfloat16_rn(v);
            else ((float*)P.y)[r * P.y_stride + c] = v;
        }
}

int launch(t0_runtime* rt, const Product& P, bool gated) {
    return P.m > 256 ? launch_pair(rt, P, gated) : launch_stream(rt, P, gated);
    const uint64_t grid = (uint64_t)ceil_div(P.m, kTile) * ceil_div(P.n, kTile);
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "m=%u, n=%u: too much for one launch", P.m, P.n);
    const DeviceGuard guard(rt->device);
    const cudaError_t e = gated ? gemm::launch_pdl(q8_gemm_kernel<true>, (uint32_t)grid, 256, 0, rt->stream, P)
                                : gemm::launch_pdl(q8_gemm_kernel<false>, (uint32_t)grid, 256, 0, rt->stream, P);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the eight-bit product failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

// What both entries check; fills `P` but for the second matrix, the bias and the activation.
int check_product(uint64_t a, uint64_t a_scales, uint32_t* a_stride, uint64_t y, uint32_t* y_stride, uint32_t m, uint32_t n, uint32_t k, bool out_bf16, Product* P) {
    memset(P, 0, sizeof *P);
    const uint32_t size = out_bf16 ? 2 : 4;
    if (k == 0) return fail(T0_ERR_INVALID, "k must be positive");
    if (k > kMaxSum) return fail(T0_ERR_UNSUPPORTED, "k=%u: sums of more than %u products may leave 32 bits", k, kMaxSum);
    if (m > 0x40000000u || n > 0x40000000u) return fail(T0_ERR_INVALID, "m=%u, n=%u: at most 2^30", m, n);
    if (m == 0 || n == 0) return T0_OK;
    int rc = check_codes("a", a, a_scales, a_stride, k);
    if (rc != T0_OK) return rc;
    if (!y) return fail(T0_ERR_INVALID, "null device pointer");
    if (y % size) return fail(T0_ERR_INVALID, "y must be aligned to its numbers");
    if (*y_stride == 0) *y_stride = n;
    if (*y_stride < n) return fail(T0_ERR_INVALID, "y: a stride of %u numbers, rows have %u", *y_stride, n);
    P->a = (const int8_t*)a; P->a_scales = (const float*)a_scales; P->y = (void*)y;
    P->a_stride = *a_stride; P->y_stride = *y_stride;
    P->m = m; P->n = n; P->k = k; P->out_bf16 = out_bf16;
    if (touch(y, (uint64_t)n * size, (uint64_t)*y_stride * size, m, a, k, *a_stride, m) || touch(y, (uint64_t)n * size, (uint64_t)*y_stride * size, m, a_scales, 4, 4, m))
        return fail(T0_ERR_INVALID, "y overlaps a or its scales");
    return T0_OK;
}

int check_weights(const char* name, uint64_t w, uint64_t scales, uint32_t* stride, int which, Product* P) {
    const uint32_t size = P->out_bf16 ? 2 : 4;
    int rc = check_codes(name, w, scales, stride, P->k);
    if (rc != T0_OK) return rc;
    if (touch((uint64_t)P->y, (uint64_t)P->n * size, P->y_stride * size, P->m, w, P->k, *stride, P->n) ||
        touch((uint64_t)P->y, (uint64_t)P->n * size, P->y_stride * size, P->m, scales, (uint64_t)P->n * 4, (uint64_t)P->n * 4, 1))
        return fail(T0_ERR_INVALID, "y overlaps %s or its scales", name);
    P->w[which] = (const int8_t*)w; P->w_scales[which] = (const float*)scales;
    P->w_stride = *stride;
    return T0_OK;
}

}  // namespace
}  // namespace q8
}  // namespace t0

using namespace t0;
using namespace t0::q8;

extern "C" {

int t0_q8_gemm(t0_runtime* rt, const t0_q8_gemm_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_gemm_args a = *args;
    Product P;
    int rc = check_product(a.a, a.a_scales, &a.a_stride, a.y, &a.y_stride, a.m, a.n, a.k, a.out_bf16 != 0, &P);
    if (rc != T0_OK) return rc;
    if (a.m == 0 || a.n == 0) return check_rt(rt);
    if ((rc = check_weights("w", a.w, a.w_scales, &a.w_stride, 0, &P)) != T0_OK) return rc;
    if (a.bias & 3) return fail(T0_ERR_INVALID, "the bias must be 4-byte aligned");
    const uint64_t size = a.out_bf16 ? 2 : 4;
    if (touch(a.y, a.n * size, a.y_stride * size, a.m, a.bias, 4ull * a.n, 4ull * a.n, 1)) return fail(T0_ERR_INVALID, "y overlaps the bias");
    P.bias = (const float*)a.bias;
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    return launch(rt, P, false);
}

int t0_q8_gated(t0_runtime* rt, const t0_q8_gated_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_gated_args a = *args;
    Product P;
    int rc = check_product(a.a, a.a_scales, &a.a_stride, a.y, &a.y_stride, a.m, a.n, a.k, a.out_bf16 != 0, &P);
    if (rc != T0_OK) return rc;
    if (a.activation != T0_TEPI_RELU && a.activation != T0_TEPI_SILU && a.activation != T0_TEPI_GELU)
        return fail(T0_ERR_INVALID, "activation=%u: relu, silu or gelu", a.activation);
    if (a.m == 0 || a.n == 0) return check_rt(rt);
    if ((rc = check_weights("gate", a.gate, a.gate_scales, &a.w_stride, 0, &P)) != T0_OK) return rc;
    if ((rc = check_weights("up", a.up, a.up_scales, &a.w_stride, 1, &P)) != T0_OK) return rc;
    P.act = a.activation;
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    return launch(rt, P, true);
}

}  // extern "C"
