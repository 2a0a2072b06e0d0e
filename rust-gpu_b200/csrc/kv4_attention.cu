// Attention over the paged four-bit key/value cache: the entry point and the kernels' choice.
#include <cmath>

#include "kv4_attention.cuh"

namespace t0 {
namespace kv4 {
namespace {

// One warp a row and query head: the tokens one after the other, running maximum and sum.
template <int D>
__global__ void __launch_bounds__(256) kv4_attention_plain_kernel(const __grid_constant__ Attention P) {
    constexpr int kPer = D / 32;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const Batch& B = P.B;
    const uint64_t unit = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
    const uint32_t lane = threadIdx.x % 32, q_heads = B.n_kv_heads * P.group, r = (uint32_t)(unit / q_heads), h = (uint32_t)(unit % q_heads);
    if (r >= B.n_rows) return;
    uint32_t b;
    Sequence s;
    if (!sequence_of_row(B, r, &b, &s)) return;
    if ((uint32_t)s.rows * P.group <= P.few) return;
    const int token = s.len - s.rows + ((int)r - s.first_row);
    const uint32_t kv_head = h / P.group;
    float q[kPer], o[kPer] = {}, m = -INFINITY, l = 0.0f;
    for (int i = 0; i < kPer; ++i) q[i] = __bfloat162float(P.q[r * P.q_stride + h * D + lane * kPer + i]);
    const int begin = P.window && token >= (int)P.window ? token - (int)P.window + 1 : 0;
    const uint32_t page_mask = (1u << B.page_log2) - 1;
    const uint8_t* block = nullptr;
    for (int j = begin; j <= token; ++j) {
        if (j == begin || ((uint32_t)j & page_mask) == 0) block = block_to_read<D>(B, b, (uint32_t)j >> B.page_log2, kv_head);
        const uint32_t slot = (uint32_t)j & page_mask;
        const uint32_t kp = *(const uint32_t*)(block + params_at<D>(B.page_log2, 0) + 4 * slot), vp = *(const uint32_t*)(block + params_at<D>(B.page_log2, 1) + 4 * slot);
        const uint32_t kw = *(const uint32_t*)(block + codes_at<D>(B.page_log2, 0) + slot * (D / 2) + lane * kPer / 8 * 4);
        const uint32_t vw = *(const uint32_t*)(block + codes_at<D>(B.page_log2, 1) + slot * (D / 2) + lane * kPer / 8 * 4);
        float dot = 0.0f;
        for (int i = 0; i < kPer; ++i) dot += q[i] * (param_step(kp) * (float)((kw >> code_shift(lane * kPer % 8 + i)) & 15) + param_low(kp));
        for (int d = 16; d; d /= 2) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
        const float x = dot * P.scale_log2, m_new = fmaxf(m, x);
        const float p = exp2_fast(x - m_new), keep = m == -INFINITY ? 0.0f : exp2_fast(m - m_new);
        m = m_new;
        l = l * keep + p;
        for (int i = 0; i < kPer; ++i) o[i] = o[i] * keep + p * (param_step(vp) * (float)((vw >> code_shift(lane * kPer % 8 + i)) & 15) + param_low(vp));
    }
    for (int i = 0; i < kPer; ++i) P.y[r * P.y_stride + h * D + lane * kPer + i] = __float2bfloat16_rn(l == 0.0f ? 0.0f : o[i] / l);
}

}  // namespace
}  // namespace kv4

size_t kv4_counter_bytes() { return kv4::kMaxCtas * sizeof(int); }

}  // namespace t0

using namespace t0;
using namespace t0::kv4;

extern "C" {

size_t t0_kv4_scratch_bytes(const t0_runtime* rt) { return rt ? kv4_counter_bytes() + kv4::decode_scratch_bytes((uint32_t)rt->sm_count) : 0; }

int t0_kv4_attention(t0_runtime* rt, const t0_kv4_batch* batch, const t0_kv4_attention_args* args) {
    Attention P;
    memset(&P, 0, sizeof P);
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    int rc = check_batch(batch, &P.B);
    if (rc != T0_OK) return rc;
    if (P.B.n_rows == 0) return check_rt(rt);
    t0_kv4_attention_args a = *args;
    const uint32_t D = batch->head_dim, width = a.n_q_heads * D;
    if (!a.q || !a.y) return fail(T0_ERR_INVALID, "null device pointer");
    if (a.n_q_heads == 0 || a.n_q_heads % batch->n_kv_heads || a.n_q_heads / batch->n_kv_heads > 64)
        return fail(T0_ERR_INVALID, "n_q_heads=%u must be a multiple of n_kv_heads=%u, at most 64 times it", a.n_q_heads, batch->n_kv_heads);
    if (!(a.scale > 0.0f) || std::isinf(a.scale)) return fail(T0_ERR_INVALID, "scale=%g must be positive and finite", (double)a.scale);
    if (a.window > 0x7FFFFFFFu) return fail(T0_ERR_INVALID, "window=%u", a.window);
    if ((rc = check_rows("q", a.q, &a.q_stride, width, 2)) != T0_OK) return rc;
    if ((rc = check_rows("y", a.y, &a.y_stride, width, 2)) != T0_OK) return rc;
    const bool in_place = a.y == a.q && (a.y_stride == a.q_stride || batch->n_rows == 1);
    if (!in_place && rows_touch(a.q, 2ull * width, 2ull * a.q_stride, a.y, 2ull * width, 2ull * a.y_stride, batch->n_rows))
        return fail(T0_ERR_INVALID, "y overlaps q (it may be q itself)");
    // the most chunks of 64 tokens that the batch may hold: the kernels count them, for every head, in 32 bits
    if ((uint64_t)batch->n_seqs * ((uint64_t)batch->table_stride * batch->page_size / 64 + 1) * batch->n_kv_heads >= 1ull << 31)
        return fail(T0_ERR_UNSUPPORTED, "%u sequences of up to %llu tokens, %u heads: too much for one call", batch->n_seqs,
                    (unsigned long long)batch->table_stride * batch->page_size, batch->n_kv_heads);
    P.q = (const __nv_bfloat16*)a.q; P.y = (__nv_bfloat16*)a.y;
    P.q_stride = a.q_stride; P.y_stride = a.y_stride;
    P.group = a.n_q_heads / batch->n_kv_heads; P.window = a.window;
    P.scale_log2 = a.scale * 1.44269504f;
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    P.B.status = rt->d_status + 1;
    P.timeout_status = rt->d_status;
    const uint64_t limit = rt->wait_limit_ns.load(std::memory_order_relaxed);
    P.wait_limit_ns = limit ? limit : ptx::kWaitLimitNs;
    if (rt->scratch_kv4.size == 0 && (rc = t0_rt_reserve_scratch(rt, T0_SCRATCH_KV4, 0)) != T0_OK) return rc;
    DeviceGuard guard(rt->device);
    P.scratch = (uint8_t*)rt->scratch_kv4.ptr;
    // Which sequences have few rows is known on the device; the host knows the most of any.
    const uint64_t columns = (uint64_t)batch->max_rows * P.group;
    P.few = P.group <= kFewColumns && (columns <= kFewColumns || batch->row_start) ? kFewColumns : 0;
    if (P.few) {
        rc = launch_decode(P, D, (uint32_t)std::min<uint64_t>(columns, kFewColumns), (uint32_t)rt->sm_count, rt->stream);
        if (rc != T0_OK) return rc;
        rt->launches.fetch_add(1);
        if (columns <= kFewColumns) return T0_OK;
    }
    const uint64_t grid = ((uint64_t)batch->n_rows * a.n_q_heads * 32 + 255) / 256;
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "too many rows and heads for one launch");
    const cudaError_t e = D == 64 ? gemm::launch_pdl(kv4_attention_plain_kernel<64>, (uint32_t)grid, 256, 0, rt->stream, P)
                                  : gemm::launch_pdl(kv4_attention_plain_kernel<128>, (uint32_t)grid, 256, 0, rt->stream, P);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "attention launch failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

}  // extern "C"
