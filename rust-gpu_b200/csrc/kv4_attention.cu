// Attention over the paged four-bit key/value cache: the entry point and the kernels' choice.
#include <cmath>

#include "kv4_attention.cuh"

namespace t0 {

size_t kv4_counter_bytes() { return kv4::kMaxCtas * sizeof(int); }

}  // namespace t0

using namespace t0;
using namespace t0::kv4;

extern "C" {

size_t t0_kv4_scratch_bytes(const t0_runtime* rt) {
    const uint32_t sms = rt ? (uint32_t)rt->sm_count : 0;
    return rt ? kv4_counter_bytes() + kv4::decode_scratch_bytes(sms) + kv4::prompt_scratch_bytes(sms) : 0;
}

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
    if (!(a.scale > 0.0f) || std::isinf(a.scale * 1.44269504f)) return fail(T0_ERR_INVALID, "scale=%g must be positive and finite, in powers of two too", (double)a.scale);
    if (a.window > 0x7FFFFFFFu) return fail(T0_ERR_INVALID, "window=%u", a.window);
    if ((rc = check_rows("q", a.q, &a.q_stride, width, 2)) != T0_OK) return rc;
    if ((rc = check_rows("y", a.y, &a.y_stride, width, 2)) != T0_OK) return rc;
    const bool in_place = a.y == a.q && (a.y_stride == a.q_stride || batch->n_rows == 1);
    if (!in_place && rows_touch(a.q, 2ull * width, 2ull * a.q_stride, a.y, 2ull * width, 2ull * a.y_stride, batch->n_rows))
        return fail(T0_ERR_INVALID, "y overlaps q (it may be q itself)");
    if ((rc = check_outside("y", batch, a.y, 2ull * width, 2ull * a.y_stride)) != T0_OK) return rc;
    // the kernels count the chunks (64 tokens for few rows, 128 against 256 rows for many) that a batch of this shape may hold, for every head, in 32 bits
    const uint64_t places = (uint64_t)batch->table_stride * batch->page_size;
    if ((uint64_t)batch->n_seqs * (places / 64 + 1) * batch->n_kv_heads >= 1ull << 31 ||
        ((uint64_t)batch->n_rows * a.n_q_heads / batch->n_kv_heads / 256 + batch->n_seqs) * (places / 128 + 4) * batch->n_kv_heads >= 1ull << 31)
        return fail(T0_ERR_UNSUPPORTED, "%u sequences of up to %llu tokens, %u heads: too much for one call", batch->n_seqs,
                    (unsigned long long)places, batch->n_kv_heads);
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
    rc = launch_prompt(P, D, (uint32_t)rt->sm_count, rt->stream);
    if (rc == T0_OK) rt->launches.fetch_add(2);
    return rc;
}

}  // extern "C"
