// The paged key/value cache in four bits: append (with the rotation of keys and queries) and read-out.
#include "gemm_common.cuh"
#include "kv4.cuh"

namespace t0 {
namespace kv4 {

int check_batch(const t0_kv4_batch* b, Batch* out) {
    if (!b) return fail(T0_ERR_INVALID, "null batch");
    if (b->page_size != 16 && b->page_size != 32 && b->page_size != 64)
        return fail(T0_ERR_UNSUPPORTED, "page_size=%u: pages hold 16, 32 or 64 tokens", b->page_size);
    if (b->head_dim != 64 && b->head_dim != 128) return fail(T0_ERR_UNSUPPORTED, "head_dim=%u: heads have 64 or 128 numbers", b->head_dim);
    if (b->n_kv_heads == 0 || b->n_kv_heads > 4096) return fail(T0_ERR_INVALID, "n_kv_heads=%u must be in 1 .. 4096", b->n_kv_heads);
    if (b->n_seqs == 0 || b->n_rows == 0) {
        *out = Batch{};
        return T0_OK;
    }
    if (b->n_seqs > (1u << 20) || b->n_rows > (1u << 24)) return fail(T0_ERR_INVALID, "%u sequences, %u rows: at most 2^20 and 2^24", b->n_seqs, b->n_rows);
    if (!b->pages || !b->page_table || !b->seq_lens) return fail(T0_ERR_INVALID, "null device pointer in the batch");
    if (b->pages & 15) return fail(T0_ERR_INVALID, "the cache must be 16-byte aligned");
    if ((b->page_table | b->seq_lens | b->row_start) & 3) return fail(T0_ERR_INVALID, "page_table, seq_lens and row_start must be 4-byte aligned");
    if (b->n_pages == 0 || b->n_pages > 0x7FFFFFFFu) return fail(T0_ERR_INVALID, "n_pages=%u", b->n_pages);
    if (b->table_stride == 0 || (uint64_t)b->table_stride * b->page_size > 0x40000000ull)
        return fail(T0_ERR_INVALID, "table_stride=%u: between one page and 2^30 tokens", b->table_stride);
    if (b->max_rows == 0 || b->max_rows > b->n_rows) return fail(T0_ERR_INVALID, "max_rows=%u must be in 1 .. n_rows=%u", b->max_rows, b->n_rows);
    if (!b->row_start && (uint64_t)b->n_seqs * b->max_rows != b->n_rows)
        return fail(T0_ERR_INVALID, "without row_start n_rows=%u must be n_seqs=%u times max_rows=%u", b->n_rows, b->n_seqs, b->max_rows);
    out->pages = (uint8_t*)b->pages;
    out->page_table = (const int32_t*)b->page_table;
    out->seq_lens = (const int32_t*)b->seq_lens;
    out->row_start = (const int32_t*)b->row_start;
    out->n_pages = b->n_pages;
    out->page_log2 = b->page_size == 16 ? 4 : b->page_size == 32 ? 5 : 6;
    out->n_kv_heads = b->n_kv_heads;
    out->n_seqs = b->n_seqs; out->table_stride = b->table_stride;
    out->n_rows = b->n_rows; out->max_rows = b->max_rows;
    return T0_OK;
}

int check_rows(const char* name, uint64_t base, uint32_t* stride, uint32_t width, uint32_t bytes) {
    if (*stride == 0) *stride = width;
    if (*stride < width) return fail(T0_ERR_INVALID, "%s: a stride of %u numbers, rows have %u", name, *stride, width);
    if ((base & 15) || (uint64_t)*stride * bytes % 16) return fail(T0_ERR_INVALID, "%s: rows must start on 16-byte boundaries", name);
    return T0_OK;
}

bool rows_touch(uint64_t a, uint64_t a_bytes, uint64_t a_stride, uint64_t b, uint64_t b_bytes, uint64_t b_stride, uint64_t rows) {
    const uint64_t a_end = a + (rows - 1) * a_stride + a_bytes, b_end = b + (rows - 1) * b_stride + b_bytes;
    if (a_end <= b || b_end <= a) return false;
    if (a_stride != b_stride || rows == 1) return true;
    const uint64_t d = b >= a ? (b - a) % a_stride : (a_stride - (a - b) % a_stride) % a_stride;       // columns of one wider array
    return d < a_bytes || d + b_bytes > a_stride;
}

int check_outside(const char* name, const t0_kv4_batch* b, uint64_t base, uint64_t bytes, uint64_t stride) {
    const uint64_t cache = b->n_pages * (uint64_t)t0_kv4_page_bytes(b->page_size, b->n_kv_heads, b->head_dim), end = base + (b->n_rows - 1) * stride + bytes;
    if (base < b->pages + cache && b->pages < end) return fail(T0_ERR_INVALID, "%s overlaps the cache", name);
    return T0_OK;
}

namespace {

struct Append {
    Batch B;
    const void *q, *k, *v;
    __nv_bfloat16* q_out;
    const float2* rope;
    const int32_t* positions;
    uint64_t q_stride, k_stride, v_stride, q_out_stride;
    uint32_t n_q_heads, n_positions, rot_dim;
    uint32_t end0, end1;                    // first pair of the second and of the third axis
    uint32_t n_axes;
    bool interleaved;
    uint32_t per_warp;                      // heads of a row that one warp takes
};

// Eight numbers as they lie in memory, and as f32: apart, so that a load is not waited for where it is issued.
template <bool F32> struct Eight { uint4 w[F32 ? 2 : 1]; };
template <bool F32>
__device__ __forceinline__ Eight<F32> load8(const void* base, uint64_t at) {
    Eight<F32> x;
    const uint4* p = (const uint4*)((const char*)base + at * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) x.w[i] = p[i];
    return x;
}
template <bool F32>
__device__ __forceinline__ void unpack8(float (&y)[8], const Eight<F32>& x) {
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            y[4 * i] = __uint_as_float(x.w[i].x); y[4 * i + 1] = __uint_as_float(x.w[i].y);
            y[4 * i + 2] = __uint_as_float(x.w[i].z); y[4 * i + 3] = __uint_as_float(x.w[i].w);
        }
    } else {
        const uint32_t u[4] = {x.w[0].x, x.w[0].y, x.w[0].z, x.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = __uint_as_float(u[i] << 16);
            y[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&p;
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// The step of a row: the smallest bf16 not below range / 15, the quotient rounded to f32.  15 b is exact for a bf16 b, and where it is not the range the two are at least a unit
// in the last place of the range apart, which is more than half a unit of the quotient: the rounded quotient is above b exactly where the range is above 15 b.  So a product
// with 1 / 15 finds the place to within a neighbour, and exact comparisons the step.
__device__ __forceinline__ float step_of(float range) {
    const int up = __float_as_int(-bf16_down(-(range * (1.0f / 15.0f))));
    float step = __int_as_float(up);
    const float below = __int_as_float(up - 0x10000);
    if (up >= 0x10000 && fmaf(-15.0f, below, range) <= 0.0f) step = below;
    if (fmaf(-15.0f, step, range) > 0.0f) step = __int_as_float(up + 0x10000);
    return step < 1.17549435e-38f ? 0.0f : step;
}
// The codes of eight numbers, packed: rint((x - low) / step), the quotient rounded to f32, for a bf16 step with `inverse` near 1 / step.  With d = x - low and c near d / step,
// d - c step is exact (a multiple of d's last place, and no larger than d); where it is not half a step it differs from half a step by more than the quotient's rounding.  So c
// is the code where that rest is below half a step; where it is not (ties are common in rows of bf16), the comparison says which neighbour is, and a tie goes to the even one.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float low, float step, float inverse) {
    const float half = 0.5f * step;
    float near[8], rest[8], worst = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float d = __fsub_rn(x[i], low);
        near[i] = fmaf(d, inverse, 12582912.0f);           // 1.5 * 2^23: the whole number in the low bits
        rest[i] = fmaf(-(near[i] - 12582912.0f), step, d);
        worst = fmaxf(worst, fabsf(rest[i]));
    }
    if (worst >= half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool odd = __float_as_uint(near[i]) & 1;
            if (rest[i] > half || (rest[i] == half && odd)) near[i] += 1.0f;
            if (rest[i] < -half || (rest[i] == -half && odd)) near[i] -= 1.0f;
            near[i] = fminf(near[i], 12582912.0f + 15.0f);
        }
    }
    uint32_t codes = 0, bias = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        codes += __float_as_uint(near[i]) << code_shift(i);
        bias += 0x4B400000u << code_shift(i);
    }
    return codes - bias;
}

// A warp takes a row, or `per_warp` of its heads where rows are few: sequence, token, page, positions and the lane's cosines and sines are found once for all of them.  A head is
// D / 8 lanes wide, eight numbers a lane, so that a warp works on several at a time and asks for the next ones before it needs them.  A lane turns its numbers, and
// either rounds them to bf16 (queries) or finds the row's range with its group and cuts them to four bits, a 32-bit word of codes a lane.  8192 rows of 32 query and
// 8 key/value heads of 128, bf16, three axes, are 181 MB (27.6 us); it takes 59.5 us, bound by its instructions (about 4400 a row, half of them the range and the codes) at the 24 warps
// an SM holds: 3 blocks of 80 registers and two loads ahead measured 71 us with the read-out behind it (now 67.4), 4 blocks 68 to 76, four loads ahead 70 (and 13 instead of 10 us at 256 rows).
// f32 rows with one axis take 64 us, 256 single tokens 7.0 and one 3.6.
template <int D, bool F32>
__global__ void __launch_bounds__(256, 3) kv4_append_kernel(const __grid_constant__ Append P) {
    constexpr uint32_t kLanes = D / 8, kAtOnce = 32 / kLanes, kAhead = 2;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const Batch& B = P.B;
    const uint32_t heads = P.n_q_heads + 2 * B.n_kv_heads, parts = (heads + P.per_warp - 1) / P.per_warp;
    const uint64_t unit = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32;
    const uint32_t lane = threadIdx.x % 32, e = lane % kLanes, sub = lane / kLanes;
    const uint32_t r = (uint32_t)(unit / parts), h0 = (uint32_t)(unit % parts) * P.per_warp, h1 = min(heads, h0 + P.per_warp);
    if (r >= B.n_rows) return;
    uint32_t b;
    Sequence s;
    if (!sequence_of_row(B, r, &b, &s)) return;
    const int token = s.len - s.rows + ((int)r - s.first_row);
    if (token < 0) return;

    // the first loads, before the chain of lookups that the turns need; each is followed by the next one to take its place
    constexpr uint32_t kSize = F32 ? 4 : 2;
    const char* const q_in = (const char*)P.q + (r * P.q_stride + 8 * e) * kSize;
    const char* const k_in = (const char*)P.k + (r * P.k_stride + 8 * e) * kSize - (uint64_t)P.n_q_heads * (D * kSize);
    const char* const v_in = (const char*)P.v + (r * P.v_stride + 8 * e) * kSize - (uint64_t)(P.n_q_heads + B.n_kv_heads) * (D * kSize);
    auto load = [&](uint32_t h) { return load8<F32>(h < P.n_q_heads ? q_in : h < P.n_q_heads + B.n_kv_heads ? k_in : v_in, h * D); };
    Eight<F32> x[kAhead];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a)
        if (h0 + a * kAtOnce + sub < h1) x[a] = load(h0 + a * kAtOnce + sub);

    // the row's positions, and the turns of the lane's numbers: (a, b) of pair i are numbers i and i + rot_dim / 2, or 2 i and 2 i + 1 of the lane itself
    float2 turn[8] = {};
    bool turns = false, second = false;
    uint32_t from = lane;                                  // the lane that has the other numbers of the pairs
    if (P.rope) {
        int pos[3] = {token, token, token};
        if (P.positions)
            for (uint32_t a = 0; a < P.n_axes; ++a) pos[a] = P.positions[(uint64_t)a * B.n_rows + r];
        bool bad = false;
        for (uint32_t a = 0; a < P.n_axes; ++a) bad |= (uint32_t)pos[a] >= P.n_positions;
        if (bad) {                                         // the row is left out as a whole, its values too
            if (lane == 0) report(B, kStatusBadPosition, r);
            return;
        }
        const uint32_t pairs = P.rot_dim / 2, away = P.rot_dim / 16;       // `away`: lanes between the two numbers of a pair
        turns = e < 2 * away;
        second = !P.interleaved && turns && e >= away;
        if (!P.interleaved && turns) from = second ? lane - away : lane + away;
        const uint32_t first_pair = P.interleaved ? 4 * e : 8 * (second ? e - away : e);
        if (turns && h0 < P.n_q_heads + B.n_kv_heads) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                if (P.interleaved && i >= 4) break;
                const uint32_t pair = first_pair + i;
                if (P.n_axes == 1) {                       // (two pairs lie on one 16-byte boundary)
                    const float4 t = *(const float4*)(P.rope + (uint64_t)pos[0] * pairs + pair);
                    turn[i] = make_float2(t.x, t.y);
                    turn[i + 1] = make_float2(t.z, t.w);
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int p = pair + j < P.end0 ? pos[0] : pair + j < P.end1 ? pos[1] : pos[2];
                        turn[i + j] = P.rope[(uint64_t)p * pairs + pair + j];
                    }
                }
            }
        }
    }
    // (first and second number of a pair differ in the sign of the sine's term alone)
    if (!P.interleaved && !second) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn[i].y = -turn[i].y;
    }
    const bool whole_turn = P.rot_dim == D;                // (the same for the whole launch: no choice lane by lane)
    auto rotate = [&](float (&y)[8]) {
        if (P.interleaved) {
            if (!turns) return;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = y[2 * i], w = y[2 * i + 1];
                y[2 * i] = __fsub_rn(__fmul_rn(u, turn[i].x), __fmul_rn(w, turn[i].y));
                y[2 * i + 1] = __fadd_rn(__fmul_rn(w, turn[i].x), __fmul_rn(u, turn[i].y));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {                       // (products and sums of pairs in one instruction would be contracted)
                const float2 other = make_float2(__shfl_sync(0xFFFFFFFFu, y[i], from), __shfl_sync(0xFFFFFFFFu, y[i + 1], from));
                const float2 z = make_float2(__fadd_rn(__fmul_rn(y[i], turn[i].x), __fmul_rn(other.x, turn[i].y)),
                                             __fadd_rn(__fmul_rn(y[i + 1], turn[i + 1].x), __fmul_rn(other.y, turn[i + 1].y)));
                if (whole_turn || turns) {
                    y[i] = z.x;
                    y[i + 1] = z.y;
                }
            }
        }
    };

    uint8_t* block = h1 > P.n_q_heads ? block_of<D>(B, b, (uint32_t)token >> B.page_log2, 0) : nullptr;
    const uint32_t slot = (uint32_t)token & ((1u << B.page_log2) - 1), block_bytes = (D + 8) << B.page_log2;
    const uint32_t group = (uint32_t)((1ull << kLanes) - 1) << (sub * kLanes), keys_end = P.n_q_heads + B.n_kv_heads;
    __nv_bfloat16* out = P.q_out + r * P.q_out_stride + 8 * e;
    for (uint32_t h = h0; h < h1; h += kAhead * kAtOnce) {
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t from_h = h + a * kAtOnce, to_h = from_h + kAtOnce, at = from_h + sub;     // the heads that the warp has now, and this lane's
            if (from_h >= h1) break;
            float y[8];
            unpack8<F32>(y, x[a]);
            if (at + kAhead * kAtOnce < h1) x[a] = load(at + kAhead * kAtOnce);
            if (P.rope && to_h <= keys_end) {
                rotate(y);
            } else if (P.rope && from_h < keys_end) {          // keys and values at once
                float z[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = y[i];
                rotate(z);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = at < keys_end ? z[i] : y[i];
            }
            if (from_h < P.n_q_heads) {
                if (at < min(h1, P.n_q_heads)) *(uint4*)(out + at * D) = pack8(y);
                if (to_h <= P.n_q_heads) continue;
            }
            if (!block) continue;
            // the range; zero times an infinity or a NaN shows it
            float mn = y[0], mx = y[0], zero = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mn = fminf(mn, y[i]);
                mx = fmaxf(mx, y[i]);
                zero = fmaf(y[i], 0.0f, zero);
            }
#pragma unroll
            for (uint32_t d = 1; d < kLanes; d *= 2) {
                mn = fminf(mn, __shfl_xor_sync(0xFFFFFFFFu, mn, d));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
            }
            bool bad = (__ballot_sync(0xFFFFFFFFu, !(zero == 0.0f)) & group) != 0;
            const float low = bf16_down(mn), range = __fsub_rn(mx, low);
            bad |= !(range < __int_as_float(0x7F800000));
            const float step = step_of(range);
            uint32_t codes = 0;
            if (!bad && step > 0.0f) {
                float inverse;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(step));
                codes = codes_of(y, low, step, inverse);
            }
            if (at >= P.n_q_heads && at < h1) {
                const uint32_t which = at < keys_end ? 0 : 1;
                uint8_t* to = block + (uint64_t)(at - (which ? keys_end : P.n_q_heads)) * block_bytes;
                *(uint32_t*)(to + codes_at<D>(B.page_log2, which) + slot * (D / 2) + 4 * e) = codes;
                if (e == 0)
                    *(uint32_t*)(to + params_at<D>(B.page_log2, which) + 4 * slot) = bad ? 0x7FC07FC0u : (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xFFFF0000u);
            }
        }
    }
}

struct Dequant {
    Batch B;
    __nv_bfloat16 *k_out, *v_out;
    uint64_t k_stride, v_stride;
    uint32_t per_warp;
};

// A warp takes a row, or `per_warp` of its 2 n_kv_heads rows of keys and values: a word of eight codes a lane, D / 8 lanes to a row, kAhead loads under way.
// A value is step * code + low rounded to bf16 in one step (value_of): a sum in f32 first, rounded again for the result, was a bf16 number off wherever f32 loses what decides a tie, and
// longer: 16 sequences of 2200 tokens on average, 8 heads of 128, are 183 MB and take 35.3 us at 5.2 TB/s (28 us at the rate of a plain copy), 38.2 in that form.  With every place worked
// out anew for a head it was 0.5 us more.
template <int D>
__global__ void __launch_bounds__(256, 5) kv4_dequant_kernel(const __grid_constant__ Dequant P) {
    constexpr uint32_t kLanes = D / 8, kAtOnce = 32 / kLanes, kAhead = 4;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const Batch& B = P.B;
    const uint32_t first = P.k_out ? 0 : B.n_kv_heads, heads = P.v_out ? 2 * B.n_kv_heads : B.n_kv_heads;      // keys, then values: those that are asked for
    const uint32_t parts = (heads - first + P.per_warp - 1) / P.per_warp;
    const uint64_t unit = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32;
    const uint32_t lane = threadIdx.x % 32, e = lane % kLanes, sub = lane / kLanes;
    const uint32_t r = (uint32_t)(unit / parts), h0 = first + (uint32_t)(unit % parts) * P.per_warp, h1 = min(heads, h0 + P.per_warp);
    if (r >= B.n_rows) return;
    uint32_t b;
    Sequence s;
    if (!sequence_of_row(B, r, &b, &s)) return;
    const int token = s.len - s.rows + ((int)r - s.first_row);
    const uint8_t* block = token < 0 ? nullptr : block_of<D>(B, b, (uint32_t)token >> B.page_log2, 0);
    if (token >= 0 && !block) return;
    const uint32_t slot = (uint32_t)token & ((1u << B.page_log2) - 1), block_bytes = (D + 8) << B.page_log2, H = B.n_kv_heads;
    // a value's places, less what its number among the heads is too large by
    const uint32_t k_codes = slot * (D / 2) + 4 * e, v_codes = codes_at<D>(B.page_log2, 1) + k_codes - H * block_bytes;
    const uint32_t k_params = params_at<D>(B.page_log2, 0) + 4 * slot, v_params = params_at<D>(B.page_log2, 1) + 4 * slot - H * block_bytes;
    __nv_bfloat16 *const k_out = P.k_out + r * P.k_stride + 8 * e, *const v_out = P.v_out + r * P.v_stride + 8 * e;
    uint32_t k128;
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(k128));
    for (uint32_t h = h0 + sub; h < h1; h += kAhead * kAtOnce) {
        uint32_t w[kAhead], p[kAhead];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t at = h + a * kAtOnce;
            w[a] = p[a] = 0;
            if (at < h1 && block) {
                w[a] = *(const uint32_t*)(block + (at * block_bytes + (at < H ? k_codes : v_codes)));
                p[a] = *(const uint32_t*)(block + (at * block_bytes + (at < H ? k_params : v_params)));
            }
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t at = h + a * kAtOnce;
            if (at >= h1) break;
            const __nv_bfloat162 step = twice(p[a] & 0xFFFFu), low = twice(p[a] >> 16);
            *(uint4*)(at < H ? k_out + at * D : v_out + (at - H) * D) =
                make_uint4(value_of(w[a], 0, k128, step, low), value_of(w[a], 1, k128, step, low), value_of(w[a], 2, k128, step, low), value_of(w[a], 3, k128, step, low));
        }
    }
}

// Head rows for one warp: all of a row's where there are warps enough without it (a few for each of the 48 or so places of an SM), else fewer.
uint32_t heads_per_warp(uint32_t rows, uint32_t heads, uint32_t at_once, uint32_t sms) {
    const uint64_t want = std::max<uint64_t>((uint64_t)rows * heads / (64ull * sms), 1);
    const uint32_t parts = (uint32_t)((heads + want - 1) / want), each = ceil_div(heads, parts);
    return ceil_div(each, at_once) * at_once;
}

}  // namespace
}  // namespace kv4

const char* kv4_status_text(int code) {
    switch (code & 0x7F000000) {
        case kStatusBadSequence: return "the length or the rows of sequence";
        case kStatusBadPage: return "a page outside the cache, of sequence";
        case kStatusBadPosition: return "a position outside the rope table, of row";
        default: return "place";
    }
}

}  // namespace t0

using namespace t0;
using namespace t0::kv4;

extern "C" {

size_t t0_kv4_page_bytes(uint32_t page_size, uint32_t n_kv_heads, uint32_t head_dim) {
    if ((page_size != 16 && page_size != 32 && page_size != 64) || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)page_size * (head_dim + 8) * n_kv_heads;
}

int t0_kv4_append(t0_runtime* rt, const t0_kv4_batch* batch, const t0_kv4_append_args* args) {
    Append P;
    memset(&P, 0, sizeof P);
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    int rc = check_batch(batch, &P.B);
    if (rc != T0_OK) return rc;
    if (P.B.n_rows == 0) return check_rt(rt);
    t0_kv4_append_args a = *args;
    const uint32_t D = batch->head_dim, size = a.in_f32 ? 4 : 2;
    if (!a.k || !a.v) return fail(T0_ERR_INVALID, "null device pointer");
    if (a.q && (!a.q_out || a.n_q_heads == 0 || a.n_q_heads > 65536)) return fail(T0_ERR_INVALID, "queries need q_out and n_q_heads (%u) in 1 .. 65536", a.n_q_heads);
    if (!a.q) a.n_q_heads = 0;
    if ((rc = check_rows("k", a.k, &a.k_stride, batch->n_kv_heads * D, size)) != T0_OK) return rc;
    if ((rc = check_rows("v", a.v, &a.v_stride, batch->n_kv_heads * D, size)) != T0_OK) return rc;
    if (a.q) {
        if ((rc = check_rows("q", a.q, &a.q_stride, a.n_q_heads * D, size)) != T0_OK) return rc;
        if ((rc = check_rows("q_out", a.q_out, &a.q_out_stride, a.n_q_heads * D, 2)) != T0_OK) return rc;
        const uint64_t q_bytes = (uint64_t)a.n_q_heads * D * size, kv_bytes = (uint64_t)batch->n_kv_heads * D * size, out_bytes = (uint64_t)a.n_q_heads * D * 2;
        const uint64_t out_stride = (uint64_t)a.q_out_stride * 2, n = batch->n_rows;
        const bool in_place = a.q_out == a.q && !a.in_f32 && (a.q_out_stride == a.q_stride || n == 1);
        if ((!in_place && rows_touch(a.q_out, out_bytes, out_stride, a.q, q_bytes, (uint64_t)a.q_stride * size, n)) ||
            rows_touch(a.q_out, out_bytes, out_stride, a.k, kv_bytes, (uint64_t)a.k_stride * size, n) ||
            rows_touch(a.q_out, out_bytes, out_stride, a.v, kv_bytes, (uint64_t)a.v_stride * size, n))
            return fail(T0_ERR_INVALID, "q_out overlaps q, k or v (it may be q itself where q is bf16)");
        if ((rc = check_outside("q_out", batch, a.q_out, out_bytes, out_stride)) != T0_OK) return rc;
    }
    if (a.rope) {
        if ((a.rope & 15) || (a.positions & 3)) return fail(T0_ERR_INVALID, "the rope table must be 16-byte aligned, positions 4-byte");
        if (a.rot_dim == 0 || a.rot_dim % 16 || a.rot_dim > D) return fail(T0_ERR_INVALID, "rot_dim=%u must be a multiple of 16, at most head_dim=%u", a.rot_dim, D);
        if (a.n_positions == 0 || a.n_positions > 0x7FFFFFFFu) return fail(T0_ERR_INVALID, "n_positions=%u", a.n_positions);
        if (a.n_axes > 3) return fail(T0_ERR_INVALID, "n_axes=%u: one to three", a.n_axes);
        if (a.n_axes <= 1) {
            if (a.n_axes == 1 && a.axis_pairs[0] && a.axis_pairs[0] != a.rot_dim / 2)
                return fail(T0_ERR_INVALID, "one axis has all %u pairs, not %u", a.rot_dim / 2, a.axis_pairs[0]);
            a.n_axes = 1;
            a.axis_pairs[0] = a.rot_dim / 2;
        } else if (!a.positions) {
            return fail(T0_ERR_INVALID, "several axes need positions");
        }
        uint64_t sum = 0;
        for (uint32_t i = 0; i < a.n_axes; ++i) sum += a.axis_pairs[i];
        if (sum != a.rot_dim / 2) return fail(T0_ERR_INVALID, "the axes have %llu pairs, rot_dim=%u", (unsigned long long)sum, a.rot_dim);
    }
    P.q = (const void*)a.q; P.k = (const void*)a.k; P.v = (const void*)a.v;
    P.q_out = (__nv_bfloat16*)a.q_out;
    P.rope = (const float2*)a.rope;
    P.positions = (const int32_t*)a.positions;
    P.q_stride = a.q_stride; P.k_stride = a.k_stride; P.v_stride = a.v_stride; P.q_out_stride = a.q_out_stride;
    P.n_q_heads = a.n_q_heads; P.n_positions = a.n_positions; P.rot_dim = a.rot_dim;
    P.n_axes = a.n_axes;
    P.interleaved = a.interleaved != 0;
    P.end0 = a.axis_pairs[0]; P.end1 = a.n_axes == 1 ? P.end0 : a.axis_pairs[0] + a.axis_pairs[1];
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    P.B.status = rt->d_status + 1;
    DeviceGuard guard(rt->device);
    const uint32_t heads = a.n_q_heads + 2 * batch->n_kv_heads;
    P.per_warp = heads_per_warp(batch->n_rows, heads, 256 / D, (uint32_t)rt->sm_count);
    const uint64_t grid = ((uint64_t)batch->n_rows * ceil_div(heads, P.per_warp) + 7) / 8;
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "too many rows and heads for one launch");
    auto go = [&](auto kernel) { return gemm::launch_pdl(kernel, (uint32_t)grid, 256, 0, rt->stream, P); };
    const cudaError_t e = D == 64 ? (a.in_f32 ? go(kv4_append_kernel<64, true>) : go(kv4_append_kernel<64, false>))
                                  : (a.in_f32 ? go(kv4_append_kernel<128, true>) : go(kv4_append_kernel<128, false>));
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "append launch failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

int t0_kv4_dequant(t0_runtime* rt, const t0_kv4_batch* batch, const t0_kv4_dequant_args* args) {
    Dequant P;
    memset(&P, 0, sizeof P);
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    int rc = check_batch(batch, &P.B);
    if (rc != T0_OK) return rc;
    if (P.B.n_rows == 0) return check_rt(rt);
    t0_kv4_dequant_args a = *args;
    const uint32_t D = batch->head_dim, width = batch->n_kv_heads * D;
    if (!a.k_out && !a.v_out) return fail(T0_ERR_INVALID, "null device pointer: neither keys nor values are asked for");
    if (a.k_out && (rc = check_rows("k_out", a.k_out, &a.k_out_stride, width, 2)) != T0_OK) return rc;
    if (a.v_out && (rc = check_rows("v_out", a.v_out, &a.v_out_stride, width, 2)) != T0_OK) return rc;
    if (a.k_out && a.v_out && rows_touch(a.k_out, 2ull * width, 2ull * a.k_out_stride, a.v_out, 2ull * width, 2ull * a.v_out_stride, batch->n_rows))
        return fail(T0_ERR_INVALID, "k_out and v_out overlap");
    if (a.k_out && (rc = check_outside("k_out", batch, a.k_out, 2ull * width, 2ull * a.k_out_stride)) != T0_OK) return rc;
    if (a.v_out && (rc = check_outside("v_out", batch, a.v_out, 2ull * width, 2ull * a.v_out_stride)) != T0_OK) return rc;
    P.k_out = (__nv_bfloat16*)a.k_out; P.v_out = (__nv_bfloat16*)a.v_out;
    P.k_stride = a.k_out_stride; P.v_stride = a.v_out_stride;
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    P.B.status = rt->d_status + 1;
    DeviceGuard guard(rt->device);
    const uint32_t heads = (a.k_out && a.v_out ? 2 : 1) * batch->n_kv_heads;
    P.per_warp = heads_per_warp(batch->n_rows, heads, 256 / D, (uint32_t)rt->sm_count);
    const uint64_t grid = ((uint64_t)batch->n_rows * ceil_div(heads, P.per_warp) + 7) / 8;
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "too many rows and heads for one launch");
    const cudaError_t e = D == 64 ? gemm::launch_pdl(kv4_dequant_kernel<64>, (uint32_t)grid, 256, 0, rt->stream, P)
                                  : gemm::launch_pdl(kv4_dequant_kernel<128>, (uint32_t)grid, 256, 0, rt->stream, P);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "read-out launch failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

}  // extern "C"
