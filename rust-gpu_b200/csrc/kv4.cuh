// The four-bit key/value cache as its kernels see it: the batch record, where a sequence's rows and tokens lie, the checks of what the
// device-side arrays hold, and the arithmetic of the codes.
#pragma once

#include <cuda_bf16.h>

#include "runtime_internal.h"

namespace t0 {
namespace kv4 {

struct Batch {
    uint8_t* pages;
    const int32_t* page_table;
    const int32_t* seq_lens;
    const int32_t* row_start;      // null: max_rows rows a sequence
    uint32_t n_pages, page_log2, n_kv_heads;
    uint32_t n_seqs, table_stride, n_rows, max_rows;
    int* status;                   // the second status word
};

// Checks what can be checked of the record on the host and fills `out`; head_dim is 64 or 128 after it.
int check_batch(const t0_kv4_batch* b, Batch* out);
// Checks the base and the stride (numbers; 0 becomes `width`) of an array of rows of `width` numbers of `bytes` bytes.
int check_rows(const char* name, uint64_t base, uint32_t* stride, uint32_t width, uint32_t bytes);
// Whether rows [a, a + a_bytes), a_stride apart, and rows of b touch; all in bytes, `rows` rows each.
bool rows_touch(uint64_t a, uint64_t a_bytes, uint64_t a_stride, uint64_t b, uint64_t b_bytes, uint64_t b_stride, uint64_t rows);
// T0_ERR_INVALID where rows that a call writes lie in the cache (all in bytes).
int check_outside(const char* name, const t0_kv4_batch* b, uint64_t base, uint64_t bytes, uint64_t stride);

// ------------------------------------------------------------------ device side
struct Sequence {
    int first_row, rows, len;      // its rows of the call and its tokens, those included; rows = 0 where it is left out
};

__device__ __forceinline__ void report(const Batch& B, int what, uint32_t index) { *(volatile int*)B.status = what | (int)(index & 0xFFFFFFu); }

// Sequence b, checked: every row it names exists and every token has a place in its row of the table.
__device__ __forceinline__ Sequence sequence(const Batch& B, uint32_t b) {
    Sequence s;
    if (B.row_start) {
        s.first_row = B.row_start[b];
        s.rows = B.row_start[b + 1] - s.first_row;
    } else {
        s.first_row = (int)(b * B.max_rows);
        s.rows = (int)B.max_rows;
    }
    s.len = B.seq_lens[b];
    const uint64_t places = (uint64_t)B.table_stride << B.page_log2;
    if (s.first_row < 0 || s.rows < 0 || (uint32_t)s.rows > B.max_rows || (uint64_t)s.first_row + (uint32_t)s.rows > B.n_rows || s.len < 0 || (uint64_t)s.len > places) {
        report(B, kStatusBadSequence, b);
        s.first_row = s.rows = s.len = 0;
    }
    return s;
}

// The sequence that row r belongs to; false where it belongs to none.  By a whole warp, with the same answer in every lane: 33 parts are told apart with one load.
__device__ __forceinline__ bool sequence_of_row(const Batch& B, uint32_t r, uint32_t* index, Sequence* s) {
    uint32_t b;
    if (B.row_start) {
        uint32_t lo = 0, hi = B.n_seqs;              // the last b with row_start[b] <= r (any index in range where the array is not ascending)
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 31) / 32, at = lo + (threadIdx.x & 31) * step;
            const uint32_t below = __popc(__ballot_sync(0xFFFFFFFFu, at < hi && (int64_t)B.row_start[at] <= (int64_t)r));
            lo += below ? (below - 1) * step : 0;
            hi = min(hi, lo + step);
        }
        b = lo;
    } else {
        b = r / B.max_rows;
    }
    *index = b;
    *s = sequence(B, b);
    return (int)r >= s->first_row && (int)r < s->first_row + s->rows;
}

// Block of (page, head); null, and reported, where the page is outside the cache.
template <int D>
__device__ __forceinline__ uint8_t* block_of(const Batch& B, uint32_t b, uint32_t table_column, uint32_t head) {
    const uint32_t page = (uint32_t)B.page_table[(uint64_t)b * B.table_stride + table_column];
    if (page >= B.n_pages) {
        report(B, kStatusBadPage, b);
        return nullptr;
    }
    return B.pages + ((uint64_t)page * B.n_kv_heads + head) * ((uint64_t)(D + 8) << B.page_log2);
}
// The same for kernels that read whole chunks: in place of a page outside the cache, page 0.
template <int D>
__device__ __forceinline__ const uint8_t* block_to_read(const Batch& B, uint32_t b, uint32_t table_column, uint32_t head) {
    const uint8_t* block = block_of<D>(B, b, table_column, head);
    return block ? block : B.pages + (uint64_t)head * ((D + 8) << B.page_log2);
}
template <int D> __device__ __forceinline__ uint32_t codes_at(uint32_t page_log2, uint32_t which) { return which * ((D / 2) << page_log2); }           // 0 keys, 1 values
template <int D> __device__ __forceinline__ uint32_t params_at(uint32_t page_log2, uint32_t which) { return (D + 4 * which) << page_log2; }

// Largest bf16 not above x, as f32.
__device__ __forceinline__ float bf16_down(float x) {
    int bits = __float_as_int(x), cut = bits & 0xFFFF0000;
    if (bits != cut && bits < 0) cut += 0x10000;
    return __int_as_float(cut);
}
// shift of code e of a word
__device__ __forceinline__ constexpr int code_shift(int e) { return 4 * ((e >> 1) + 4 * (e & 1)); }

__device__ __forceinline__ float param_step(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float param_low(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

// step * code + low, rounded once, of nibbles i and i + 4: 128 + code in a bf16, less 128, times step plus low
__device__ __forceinline__ uint32_t value_of(uint32_t w, int i, uint32_t k128, __nv_bfloat162 step, __nv_bfloat162 low) {
    uint32_t x;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(x) : "r"(w >> (4 * i)), "r"(k128));
    const __nv_bfloat162 k = __nv_bfloat162(__ushort_as_bfloat16(0x4300), __ushort_as_bfloat16(0x4300));
    const __nv_bfloat162 v = __hfma2(__hsub2(*(const __nv_bfloat162*)&x, k), step, low);
    return *(const uint32_t*)&v;
}
__device__ __forceinline__ __nv_bfloat162 twice(uint32_t bits16) {
    const uint32_t x = bits16 * 0x10001u;
    return *(const __nv_bfloat162*)&x;
}

}  // namespace kv4
}  // namespace t0
