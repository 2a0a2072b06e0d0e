// Rows in eight bits as the kernels of the integer products see them, and what their entries check.
#pragma once

#include <cuda_bf16.h>

#include <cuda.h>

#include "gemm_common.cuh"
#include "kv4.cuh"

namespace t0 {
namespace q8 {

constexpr uint32_t kMaxRowDim = 32768;     // rows that are made eight bits: what the largest block of threads holds in registers
constexpr uint32_t kMaxSum = 131071;       // terms of 128 * 128 at most that an i32 holds

// One product or one gated pair (w[1], w_scales[1]: the second matrix).
struct Product {
    const int8_t* a;
    const float* a_scales;
    const int8_t* w[2];
    const float* w_scales[2];
    const float* bias;
    void* y;
    uint64_t a_stride, w_stride, y_stride;
    uint32_t m, n, k;
    uint32_t act;                          // T0_TEPI_*, gated pairs only
    bool out_bf16;
};

// Checks the codes and scales of an array of rows; a stride of 0 becomes the length rounded up to 16.
int check_codes(const char* name, uint64_t codes, uint64_t scales, uint32_t* stride, uint32_t length);
// Whether rows of `a` and rows of `b` touch, all in bytes.
bool touch(uint64_t a, uint64_t a_bytes, uint64_t a_stride, uint64_t a_rows, uint64_t b, uint64_t b_bytes, uint64_t b_stride, uint64_t b_rows);

// The kernels: what each is for stands with it.
int launch_pair(t0_runtime* rt, const Product& P, bool gated);
// How the stream kernel cuts a product: rows of the weights and tokens to a tile, parts of K (four at most); parts = 0: pairs take it.
struct Cut { uint32_t rows, tokens, parts; };
constexpr uint32_t kMostTokens = 256;      // of a tile, both products' together
int launch_stream(t0_runtime* rt, const Product& P, bool gated, const Cut& cut);

// Box of 128 codes of `box_rows` rows, 128-byte swizzle; codes from `length` on and rows from `rows` on are read as zero.
int make_map_codes(CUtensorMap* map, const int8_t* codes, uint64_t stride, uint32_t rows, uint32_t length, uint32_t box_rows);

#ifdef __CUDACC__
// Two f32 in one register pair: the adders and multipliers take both at once, each rounded by itself.
__device__ __forceinline__ uint64_t pair_of(float2 a) {
    uint64_t x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    return x;
}
__device__ __forceinline__ float2 two_of(uint64_t x) {
    float2 a;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(x));
    return a;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)));
    return two_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a)), "l"(pair_of(b)));
    return two_of(d);
}
// The gate's act, in place.  f32 rows: as the epilogues of the same names compute it.  bf16 rows: x / (1 + 2^(slope x)) by the hardware's power of two (within 2^-22 of its value) and reciprocal
// (2^-23) as they come, which is far below half a step of bf16 (the step of Newton's method that f32 rows take more: gated 100 x 14336 x 4096 of f32 24.3 us without it, 24.5 so).  Either way on a quarter of 1 + 2^(slope x), so that neither that nor its
// reciprocal leaves the normal range before the power reaches 2^128, from where on the sigmoid is zero.
template <int kCount>
__device__ __forceinline__ void gate(float (&v)[kCount], uint32_t act, bool out_bf16) {
    if (act == T0_TEPI_RELU) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];         // (NaN stays)
    } else if (out_bf16) {
        const float slope = act == T0_TEPI_GELU ? -1.702f * 1.44269504088896340736f : -1.44269504088896340736f;
#pragma unroll
        for (int j = 0; j < kCount; j += 2) {
            float e[2], r[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i]) : "f"(__fmaf_rn(v[j + i], slope, -2.0f)));
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r[i]) : "f"(e[i] + 0.25f));
            }
            const float2 x = mul2(mul2(make_float2(v[j], v[j + 1]), make_float2(0.25f, 0.25f)), make_float2(r[0], r[1]));
            v[j] = x.x, v[j + 1] = x.y;
        }
    } else {
        const float times = act == T0_TEPI_GELU ? 1.702f : 1.0f;
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] *= gemm::sigmoid_seq(v[j] * times);
    }
}
// exact sums as y has them, but for the bias: three roundings
__device__ __forceinline__ float2 scaled(int32_t sum0, int32_t sum1, float2 a_scale, float2 w_scale) {
    return mul2(mul2(make_float2(__int2float_rn(sum0), __int2float_rn(sum1)), a_scale), w_scale);
}
#endif

}  // namespace q8
}  // namespace t0
