// Rows in eight bits as the kernels of the integer products see them, and what their entries check.
#pragma once

#include <cuda_bf16.h>

#include <cuda.h>

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
// How the stream kernel cuts a product: rows of the weights and tokens to a tile, parts of K; parts = 0: pairs take it.
struct Cut { uint32_t rows, tokens, parts; };
constexpr uint32_t kMostTokens = 256;      // of a tile, both products' together
int launch_stream(t0_runtime* rt, const Product& P, bool gated, const Cut& cut);

// Box of 128 codes of `box_rows` rows, 128-byte swizzle; codes from `length` on and rows from `rows` on are read as zero.
int make_map_codes(CUtensorMap* map, const int8_t* codes, uint64_t stride, uint32_t rows, uint32_t length, uint32_t box_rows);

#ifdef __CUDACC__
__device__ __forceinline__ float sigmoid(float x) {
    // 1 / (1 + 2^(-x log2 e)): the hardware's power of two and reciprocal, and one step of Newton's method for the quotient; on d / 4, so that neither d nor the result leaves the
    // normal range before d overflows, from where on the result is zero.
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504088896340736f));
    const float d = __fmaf_rn(e, 0.25f, 0.25f);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = __fmaf_rn(r, __fmaf_rn(-d, r, 1.0f), r) * 0.25f;
    return d <= 0x1p126f ? r : d != d ? d : 0.0f;
}
__device__ __forceinline__ float activate(float x, uint32_t act) {
    return act == T0_TEPI_RELU ? (x < 0.0f ? 0.0f : x) : x * sigmoid(act == T0_TEPI_GELU ? x * 1.702f : x);
}
// the exact sum as y has it, but for the bias: three roundings
__device__ __forceinline__ float scaled(int32_t sum, float a_scale, float w_scale) { return __fmul_rn(__fmul_rn(__int2float_rn(sum), a_scale), w_scale); }
#endif

}  // namespace q8
}  // namespace t0
