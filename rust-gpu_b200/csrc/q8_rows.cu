// Rows into eight bits with a scale for each, and the way back.
#include "q8_rows.cuh"

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

int check_dim(uint32_t rows, uint32_t dim, uint32_t most) {
    if (dim == 0 || dim > most) return fail(dim ? T0_ERR_UNSUPPORTED : T0_ERR_INVALID, "dim=%u: 1 .. %u", dim, most);
    if (rows > 0x7FFFFFFFu) return fail(T0_ERR_INVALID, "n_rows=%u", rows);
    return T0_OK;
}

int finish_rows(t0_runtime* rt, cudaError_t e) {
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the rows in eight bits failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

namespace {

struct Back {
    const int8_t* q;
    const float* scales;
    void* y;
    uint64_t q_stride, y_stride;
    uint64_t chunks;                                   // of all rows
    uint32_t dim, per_row, magic;                      // chunks a row; 2^32 / per_row, rounded up
};

// Eight codes a chunk, so that a warp's stores stand side by side, and four chunks a thread, asked for together: 1024 chunks a block, whatever rows they are of.
// Bound by memory: 8192 x 14336 to bf16 55.3 us (6.4 TB/s), 8192 x 4096 17.2 (5.9; 20.1 with sixteen codes a thread).
template <bool kOutF32>
__global__ void __launch_bounds__(256) q8_dequant_kernel(const Back P) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const uint64_t first = (uint64_t)blockIdx.x * 1024, row0 = first / P.per_row;
    const uint32_t skip = (uint32_t)(first - row0 * P.per_row);
    uint2 w[4];
    float scale[4];
    uint64_t row[4];
    uint32_t at[4], have[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        // the row of a chunk: x < per_row + 1024, for which the product with the rounded inverse is exact
        const uint32_t x = skip + c * 256 + threadIdx.x, r = P.per_row == 1 ? x : __umulhi(x, P.magic);
        row[c] = row0 + r;
        at[c] = (x - r * P.per_row) * 8;
        have[c] = first + c * 256 + threadIdx.x < P.chunks ? P.dim - at[c] : 0;
        w[c] = make_uint2(0, 0);
        scale[c] = 0.0f;
        if (!have[c]) continue;
        w[c] = *(const uint2*)(P.q + row[c] * P.q_stride + at[c]);     // (a row's last chunk with what lies behind it, up to the stride)
        scale[c] = P.scales[row[c]];
    }
    const float2 k = make_float2(-8388736.0f, -8388736.0f);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (!have[c]) break;
        const float2 scale2 = make_float2(scale[c], scale[c]);
        float2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {                  // code + 128 in the low bits of 2^23, less 2^23 + 128: exact, and not the conversion's eighth of the adder's rate
            const uint32_t u = (i < 2 ? w[c].x : w[c].y) ^ 0x80808080u;
            v[i] = mul2(add2(make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + 2 * (i & 1))), __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7541 + 2 * (i & 1)))), k), scale2);
        }
        store8<kOutF32>((char*)P.y + row[c] * P.y_stride * (kOutF32 ? 4 : 2), at[c], have[c], v);
    }
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
    prepare_rows(rt, P);
    const DeviceGuard guard(rt->device);
    return finish_rows(rt, P.x_f32 ? launch_by_dim<false, true, kNone>(rt, P) : launch_by_dim<false, false, kNone>(rt, P));
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
    P.q_stride = a.q_stride; P.y_stride = a.y_stride; P.dim = a.dim; P.per_row = ceil_div(a.dim, 8);
    P.magic = (uint32_t)(((1ull << 32) + P.per_row - 1) / P.per_row);
    P.chunks = n * P.per_row;
    const uint64_t grid = (P.chunks + 1023) / 1024;
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "too many rows for one launch");
    const DeviceGuard guard(rt->device);
    const cudaError_t e = a.out_f32 ? gemm::launch_pdl(q8_dequant_kernel<true>, (uint32_t)grid, 256, 0, rt->stream, P) : gemm::launch_pdl(q8_dequant_kernel<false>, (uint32_t)grid, 256, 0, rt->stream, P);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the read-out failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

}  // extern "C"
