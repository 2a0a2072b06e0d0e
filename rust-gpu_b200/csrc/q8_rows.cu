// Rows into eight bits with a scale for each, the root-mean-square norm that leaves such rows, and the way back.
//
// A row is read once and stays in its threads' registers between the two passes over it (its largest number, or for the norm the sum of its squares and then its largest
// number; the codes).  What bounds these kernels is memory: a row's bytes in and out.
#include <cmath>

#include "gemm_common.cuh"
#include "q8.cuh"
#include "runtime_internal.h"

namespace t0 {
namespace q8 {

int check_codes(const char* name, uint64_t codes, uint64_t scales, uint32_t* stride, uint32_t length) {
    if (!codes || !scales) return fail(T0_ERR_INVALID, "null device pointer: %s needs codes and scales", name);
    if (codes & 15 || scales & 3) return fail(T0_ERR_INVALID, "%s: codes must be 16-byte aligned, scales 4-byte", name);
    if (*stride == 0) *stride = (length + 15) & ~15u;
    if (*stride % 16 || *stride < length) return fail(T0_ERR_INVALID, "%s: a stride of %u must be a multiple of 16, at least %u", name, *stride, length);
    return T0_OK;
}

bool touch(uint64_t a, uint64_t a_bytes, uint64_t a_stride, uint64_t a_rows, uint64_t b, uint64_t b_bytes, uint64_t b_stride, uint64_t b_rows) {
    if (!a || !b || !a_rows || !b_rows) return false;
    if (a + (a_rows - 1) * a_stride + a_bytes <= b || b + (b_rows - 1) * b_stride + b_bytes <= a) return false;
    if (a_stride != b_stride) return true;
    const uint64_t d = b >= a ? (b - a) % a_stride : (a_stride - (a - b) % a_stride) % a_stride;       // columns of one wider array
    return d < a_bytes || d + b_bytes > a_stride;
}

namespace {

struct Rows {
    const void *x, *residual, *weight;
    void* residual_out;
    int8_t* q;
    float* scales;
    __nv_bfloat16* y;
    uint64_t x_stride, residual_stride, residual_out_stride, q_stride, y_stride;
    uint32_t n_rows, dim;
    double inv_dim, eps;
    bool x_f32, residual_f32, weight_f32;
};

// Eight numbers from `at` on, as f32; those from `end` on are zero.
__device__ __forceinline__ void load8(float (&v)[8], const void* base, uint64_t at, uint32_t have, bool f32) {
    if (have >= 8) {
        if (f32) {
            const float4 a = ((const float4*)((const float*)base + at))[0], b = ((const float4*)((const float*)base + at))[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 w = *(const uint4*)((const uint16_t*)base + at);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = i >= (int)have ? 0.0f : f32 ? ((const float*)base)[at + i] : __uint_as_float((uint32_t)((const uint16_t*)base)[at + i] << 16);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&p;
}
__device__ __forceinline__ void store8(void* base, uint64_t at, uint32_t have, bool f32, const float (&v)[8]) {
    if (have >= 8) {
        if (f32) {
            float4* p = (float4*)((float*)base + at);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *(uint4*)((uint16_t*)base + at) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < (int)have) {
            if (f32) ((float*)base)[at + i] = v[i];
            else ((__nv_bfloat16*)base)[at + i] = __float2bfloat16_rn(v[i]);
        }
}

// kThreads threads a row, eight numbers a chunk, kChunks chunks a thread; rows of one warp share a block.
template <int kThreads, int kChunks, bool kNorm>
__global__ void __launch_bounds__(kThreads == 32 ? 256 : kThreads) q8_rows_kernel(const Rows P) {
    constexpr int kWarps = kThreads / 32;
    __shared__ double sums[kNorm && kWarps > 1 ? kWarps : 1];
    __shared__ uint32_t tops[kWarps > 1 ? kWarps : 1];
    const uint32_t t = kWarps == 1 ? threadIdx.x & 31 : threadIdx.x, warp = t >> 5;
    const uint64_t row = kWarps == 1 ? (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    if (row >= P.n_rows) return;                       // whole warps, and only where a block has no barriers
    float v[kChunks][8];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const uint32_t e = (c * kThreads + t) * 8;
        load8(v[c], P.x, row * P.x_stride + e, e < P.dim ? P.dim - e : 0, P.x_f32);
    }
    if constexpr (kNorm) {
        if (P.residual) {
            float u[kChunks][8];
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8;
                load8(u[c], P.residual, row * P.residual_stride + e, e < P.dim ? P.dim - e : 0, P.residual_f32);
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[c][i] = __fadd_rn(v[c][i], u[c][i]);
                    if (!P.residual_f32) v[c][i] = __bfloat162float(__float2bfloat16_rn(v[c][i]));
                }
                if (P.residual_out && e < P.dim) store8(P.residual_out, row * P.residual_out_stride + e, P.dim - e, P.residual_f32, v[c]);
            }
        }
        double sum = 0;                                // squares of f32 are exact in f64
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fma((double)v[c][i], (double)v[c][i], sum);
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        if constexpr (kWarps > 1) {
            if ((t & 31) == 0) sums[warp] = sum;
            __syncthreads();
            sum = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) sum += sums[w];
        }
        const float r = (float)rsqrt(fma(sum, P.inv_dim, P.eps));
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const uint32_t e = (c * kThreads + t) * 8;
            if (e >= P.dim) continue;
            float w[8];
            load8(w, P.weight, e, P.dim - e, P.weight_f32);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = __fmul_rn(__fmul_rn(v[c][i], r), w[i]);
            if (P.dim - e < 8) {                       // what lies behind the row stays zero, whatever r is
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = i < (int)(P.dim - e) ? v[c][i] : 0.0f;
            }
            if (P.y) store8(P.y, row * P.y_stride + e, P.dim - e, false, v[c]);
        }
        if (!P.q) return;
    }
    // the largest of the row: the bits of sizes are in their order, infinities and NaNs above all numbers
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[c][i]) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if constexpr (kWarps > 1) {
        if ((t & 31) == 0) tops[warp] = top;
        __syncthreads();
        top = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = max(top, tops[w]);
    }
    const float most = __uint_as_float(top);
    const bool held = most >= 0x1p-119f && top < 0x7F800000u;
    const float inverse = held ? __fdiv_rn(127.0f, most) : 0.0f;
    if (t == 0) P.scales[row] = held ? __fdiv_rn(most, 127.0f) : top < 0x7F800000u ? 0.0f : __uint_as_float(0x7FFFFFFFu);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const uint32_t e = (c * kThreads + t) * 8;
        if (e >= P.dim) continue;
        uint32_t w[2] = {0, 0};
        if (held) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i >> 2] |= ((uint32_t)__float2int_rn(__fmul_rn(v[c][i], inverse)) & 0xFFu) << (8 * (i & 3));
        }
        int8_t* q = P.q + row * P.q_stride + e;
        if (P.dim - e >= 8) {
            *(uint2*)q = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < (int)(P.dim - e)) q[i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
    }
}

template <bool kNorm>
int launch_rows(t0_runtime* rt, const Rows& P) {
    const DeviceGuard guard(rt->device);
    // the fewest threads that hold the row in two chunks (registers for four rows or more an SM); above 8192, and in single warps, in four
    const auto go = [&](auto kernel, uint32_t threads) {
        return gemm::launch_pdl(kernel, threads == 32 ? (uint32_t)(((uint64_t)P.n_rows + 7) / 8) : P.n_rows, threads == 32 ? 256u : threads, 0, rt->stream, P);
    };
    const cudaError_t e = P.dim <= 1024 ? go(q8_rows_kernel<32, 4, kNorm>, 32) : P.dim <= 2048 ? go(q8_rows_kernel<128, 2, kNorm>, 128)
                        : P.dim <= 4096 ? go(q8_rows_kernel<256, 2, kNorm>, 256) : P.dim <= 8192 ? go(q8_rows_kernel<512, 2, kNorm>, 512)
                        : P.dim <= 16384 ? go(q8_rows_kernel<512, 4, kNorm>, 512) : go(q8_rows_kernel<1024, 4, kNorm>, 1024);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the rows in eight bits failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

struct Back {
    const int8_t* q;
    const float* scales;
    void* y;
    uint64_t q_stride, y_stride;
    uint32_t dim, parts;                               // blocks a row
    bool out_f32;
};

// Sixteen codes a thread, 4096 a block.
__global__ void __launch_bounds__(256) q8_dequant_kernel(const Back P) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint64_t row = blockIdx.x / P.parts;
    const uint32_t e = ((blockIdx.x % P.parts) * 256 + threadIdx.x) * 16;
    if (e >= P.dim) return;
    const float scale = P.scales[row];
    const int8_t* q = P.q + row * P.q_stride + e;
    uint32_t w[4] = {0, 0, 0, 0};
    const uint32_t have = P.dim - e;
    if (have >= 16) {
        const uint4 u = *(const uint4*)q;
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < (int)have) w[i >> 2] |= (uint32_t)(uint8_t)q[i] << (8 * (i & 3));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn((float)(int8_t)(w[2 * h + (i >> 2)] >> (8 * (i & 3))), scale);
        if (have > (uint32_t)(8 * h)) store8(P.y, row * P.y_stride + e + 8 * h, have - 8 * h, P.out_f32, v);
    }
}

int check_dim(uint32_t rows, uint32_t dim, uint32_t most) {
    if (dim == 0 || dim > most) return fail(dim ? T0_ERR_UNSUPPORTED : T0_ERR_INVALID, "dim=%u: 1 .. %u", dim, most);
    if (rows > 0x7FFFFFFFu) return fail(T0_ERR_INVALID, "n_rows=%u", rows);
    return T0_OK;
}

}  // namespace
}  // namespace q8
}  // namespace t0

using namespace t0;
using namespace t0::q8;

extern "C" {

int t0_q8_quant(t0_runtime* rt, const t0_q8_quant_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_quant_args a = *args;
    const uint32_t size = a.x_f32 ? 4 : 2;
    int rc = check_dim(a.n_rows, a.dim, kMaxRowDim);
    if (rc != T0_OK) return rc;
    if (a.n_rows == 0) return check_rt(rt);
    if (!a.x) return fail(T0_ERR_INVALID, "null device pointer");
    if ((rc = kv4::check_rows("x", a.x, &a.x_stride, a.dim, size)) != T0_OK) return rc;
    if ((rc = check_codes("q", a.q, a.scales, &a.q_stride, a.dim)) != T0_OK) return rc;
    const uint64_t x_bytes = (uint64_t)a.dim * size, x_step = (uint64_t)a.x_stride * size, n = a.n_rows;
    if (touch(a.q, a.dim, a.q_stride, n, a.x, x_bytes, x_step, n) || touch(a.scales, 4, 4, n, a.x, x_bytes, x_step, n) || touch(a.scales, 4, 4, n, a.q, a.dim, a.q_stride, n))
        return fail(T0_ERR_INVALID, "q, scales and x overlap");
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    Rows P;
    memset(&P, 0, sizeof P);
    P.x = (const void*)a.x; P.q = (int8_t*)a.q; P.scales = (float*)a.scales;
    P.x_stride = a.x_stride; P.q_stride = a.q_stride;
    P.n_rows = a.n_rows; P.dim = a.dim; P.x_f32 = a.x_f32 != 0;
    return launch_rows<false>(rt, P);
}

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
    P.x = (const void*)a.x; P.residual = (const void*)a.residual; P.weight = (const void*)a.weight; P.residual_out = (void*)a.residual_out;
    P.q = (int8_t*)a.q; P.scales = (float*)a.scales; P.y = (__nv_bfloat16*)a.y;
    P.x_stride = a.x_stride; P.residual_stride = a.residual_stride; P.residual_out_stride = a.residual_out_stride; P.q_stride = a.q_stride; P.y_stride = a.y_stride;
    P.n_rows = a.n_rows; P.dim = a.dim;
    P.inv_dim = 1.0 / a.dim; P.eps = a.eps;
    P.x_f32 = a.x_f32 != 0; P.residual_f32 = a.residual_f32 != 0; P.weight_f32 = a.weight_f32 != 0;
    return launch_rows<true>(rt, P);
}

int t0_q8_dequant(t0_runtime* rt, const t0_q8_dequant_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_dequant_args a = *args;
    const uint32_t size = a.out_f32 ? 4 : 2;
    int rc = check_dim(a.n_rows, a.dim, kMaxSum);
    if (rc != T0_OK) return rc;
    if (a.n_rows == 0) return check_rt(rt);
    if (!a.y) return fail(T0_ERR_INVALID, "null device pointer");
    if ((rc = check_codes("q", a.q, a.scales, &a.q_stride, a.dim)) != T0_OK) return rc;
    if ((rc = kv4::check_rows("y", a.y, &a.y_stride, a.dim, size)) != T0_OK) return rc;
    const uint64_t y_bytes = (uint64_t)a.dim * size, y_step = (uint64_t)a.y_stride * size, n = a.n_rows;
    if (touch(a.y, y_bytes, y_step, n, a.q, a.dim, a.q_stride, n) || touch(a.y, y_bytes, y_step, n, a.scales, 4, 4, n)) return fail(T0_ERR_INVALID, "y overlaps q or scales");
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    Back P;
    P.q = (const int8_t*)a.q; P.scales = (const float*)a.scales; P.y = (void*)a.y;
    P.q_stride = a.q_stride; P.y_stride = a.y_stride; P.dim = a.dim; P.parts = ceil_div(a.dim, 4096); P.out_f32 = a.out_f32 != 0;
    const uint64_t grid = n * P.parts;
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "too many rows for one launch");
    const DeviceGuard guard(rt->device);
    const cudaError_t e = gemm::launch_pdl(q8_dequant_kernel, (uint32_t)grid, 256, 0, rt->stream, P);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the read-out failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

}  // extern "C"
