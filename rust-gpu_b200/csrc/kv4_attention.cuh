// What the attention kernels over the four-bit cache share.
#pragma once

#include "gemm_common.cuh"
#include "kv4.cuh"

namespace t0 {
namespace kv4 {

struct Attention {
    Batch B;
    const __nv_bfloat16* q;
    __nv_bfloat16* y;
    uint64_t q_stride, y_stride;
    uint32_t group;                // query heads to a key/value head
    uint32_t window;               // 0 = all
    float scale_log2;              // scale * log2(e): scores are powers of two here
    uint32_t few;                  // a sequence with at most this many rows x group is the kv4_decode kernel's
    int* timeout_status;           // the first status word
    uint64_t wait_limit_ns;
    uint8_t* scratch;
};

// rows x group that kv4_decode takes: what its registers hold (two column tiles of eight).  131072 tokens of 8 heads of 128 (143 MB), and 32 times 4096: 44 and 43 us up to 8 columns, 55 up to 16
// there; 133 and 120 from 17 to 64 in kv4_prompt, which makes 128 rows of any number.
constexpr uint32_t kFewColumns = 16;
constexpr uint32_t kMaxCtas = 160;                       // of a persistent launch, one for each SM: arrival counters, parts of one item

size_t decode_scratch_bytes(uint32_t sms);               // behind the counters
size_t prompt_scratch_bytes(uint32_t sms);
int launch_prompt(const Attention& p, uint32_t head_dim, uint32_t sms, cudaStream_t stream);      // two kernels
int launch_decode(const Attention& p, uint32_t head_dim, uint32_t columns, uint32_t sms, cudaStream_t stream);

// First token that any row of the sequence sees.
__device__ __forceinline__ int first_seen(const Sequence& s, uint32_t window) {
    const int p = s.len - s.rows;
    return window && p >= (int)window ? p - (int)window + 1 : 0;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace kv4
}  // namespace t0
