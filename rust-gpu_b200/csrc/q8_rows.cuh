// Rows into eight bits with a scale for each, the root-mean-square norm that leaves such rows, and the way back.
//
// A row is read once and stays in its threads' registers between the two passes over it (its largest number, or for the norm the sum of its squares and then its largest
// number; the codes).  What bounds these kernels is memory, a row's bytes in and out, and with the norm the issue of instructions beside it: 8192 x 14336 of bf16 into eight bits 56.4 us (6.2 TB/s, 95 %
// of a plain copy's rate), the norm with residual of 8192 x 4096 of bf16 41.4 us (5.7 TB/s, 69 % of issue; a thread's fixed work is half of it).
#pragma once

#include <cmath>

#include "gemm_common.cuh"
#include "q8.cuh"
#include "runtime_internal.h"

namespace t0 {
namespace q8 {

constexpr uint32_t kMostSlots = 16;
constexpr uint32_t kMostRing = 220u << 10;             // shared memory that a ring may have; what a block has beside it is a few hundred bytes

struct Rows {
    const void *x, *residual, *weight;
    void* residual_out;
    int8_t* q;
    float* scales;
    __nv_bfloat16* y;
    uint64_t x_stride, residual_stride, residual_out_stride, q_stride, y_stride;
    uint32_t n_rows, dim;
    uint32_t slots, slot_bytes, residual_at;           // the ring: rows, bytes a row, where in it the residual begins
    uint32_t drop_load;
    int* status;
    uint64_t wait_limit_ns;
    double inv_dim, eps;
    bool x_f32, residual_f32, weight_f32;
};

// The launch for one type of x; each is a translation unit's.
cudaError_t launch_norm_bf16(t0_runtime* rt, Rows& P);
cudaError_t launch_norm_f32(t0_runtime* rt, Rows& P);
// What all of them do first; the caller holds the device.
inline void prepare_rows(t0_runtime* rt, Rows& P) {
    P.status = rt->d_status;
    const uint64_t limit = rt->wait_limit_ns.load(std::memory_order_relaxed);
    P.wait_limit_ns = limit ? limit : ptx::kWaitLimitNs;
}
int check_dim(uint32_t rows, uint32_t dim, uint32_t most);
int finish_rows(t0_runtime* rt, cudaError_t e);        // the call's answer, from the launch's

namespace {

// The largest of a and of two sizes; NaN where one is.
__device__ __forceinline__ float most_of(float a, float2 b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(fabsf(b.x)), "f"(fabsf(b.y)));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float2 a) {
    const __nv_bfloat162 p = __float22bfloat162_rn(a);
    return *(const uint32_t*)&p;
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }

// Eight numbers from element `at` of a row on; of the last ones of the row only `have`, the others zero.
template <bool kF32>
__device__ __forceinline__ void load8(float2 (&v)[4], const void* row, uint32_t at, uint32_t have) {
    if (have >= 8) {
        const uint4* p = (const uint4*)((const char*)row + at * (kF32 ? 4 : 2));
        const uint4 a = p[0];
        if constexpr (kF32) {
            const uint4 b = p[1];
            v[0] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y)); v[1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
            v[2] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y)); v[3] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
        } else {
            v[0] = unpack_bf16(a.x); v[1] = unpack_bf16(a.y); v[2] = unpack_bf16(a.z); v[3] = unpack_bf16(a.w);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = i >= (int)have ? 0.0f : kF32 ? ((const float*)row)[at + i] : __uint_as_float((uint32_t)((const uint16_t*)row)[at + i] << 16);
        if (i & 1) v[i >> 1].y = f;
        else v[i >> 1].x = f;
    }
}
// ... from shared memory, whole.
template <bool kF32>
__device__ __forceinline__ void lds8(float2 (&v)[4], uint32_t at) {
    uint32_t a[4], b[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at) : "memory");
    if constexpr (kF32) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(at + 16) : "memory");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v[i] = make_float2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1]));
            v[2 + i] = make_float2(__uint_as_float(b[2 * i]), __uint_as_float(b[2 * i + 1]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = unpack_bf16(a[i]);
    }
}
template <bool kF32>
__device__ __forceinline__ void store8(void* row, uint32_t at, uint32_t have, const float2 (&v)[4]) {
    if (have >= 8) {
        uint4* p = (uint4*)((char*)row + at * (kF32 ? 4 : 2));
        if constexpr (kF32) {
            p[0] = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
            p[1] = make_uint4(__float_as_uint(v[2].x), __float_as_uint(v[2].y), __float_as_uint(v[3].x), __float_as_uint(v[3].y));
        } else {
            p[0] = make_uint4(pack_bf16(v[0]), pack_bf16(v[1]), pack_bf16(v[2]), pack_bf16(v[3]));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < (int)have) {
            const float f = i & 1 ? v[i >> 1].y : v[i >> 1].x;
            if constexpr (kF32) ((float*)row)[at + i] = f;
            else ((__nv_bfloat16*)row)[at + i] = __float2bfloat16_rn(f);
        }
}
// Four whole numbers of at most 127 in size, halves rounded to even, as bytes: 1.5 * 2^23 is added, which leaves the number in the low bits of the sum (the conversion instruction
// has an eighth of the adder's rate).  One at a time: the assembler makes one operation of a product and a sum of pairs, which loses the product's rounding and with it the ties.
__device__ __forceinline__ uint32_t bytes_of(float2 a, float2 b) {
    const float k = 12582912.0f;
    const uint32_t x = __float_as_uint(__fadd_rn(a.x, k)), y = __float_as_uint(__fadd_rn(a.y, k)), z = __float_as_uint(__fadd_rn(b.x, k)), w = __float_as_uint(__fadd_rn(b.y, k));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// 1 / sqrt(m) to f64's last places: the hardware's f32 estimate (2^-22) and one cubic step, 1 - m r^2 = e, r (1 + e / 2 + 3 e^2 / 8); outside of f32's range the library's function.
__device__ __forceinline__ double inverse_root(double m) {
    const float f = (float)m;
    if (!(f > 1e-30f && f < 1e30f)) return rsqrt(m);
    float r0;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(f));
    const double r = r0, e = fma(-m * r, r, 1.0);
    return fma(r * e, fma(e, 0.375, 0.5), r);
}

enum { kNone = 0, kBf16 = 1, kF32 = 2 };               // the residual's type

// What a warp that has given up on a row leaves in the place of its sum of squares, or of its largest size: neither is ever one.  (With a sum of minus infinity among them the mean is that or NaN, so
// that only rows of next to nothing and of NaNs look for it.)
constexpr double kGone = -HUGE_VAL;
constexpr uint32_t kGoneTop = 0xFFFFFFFFu;

// Rows of up to kThreads * kChunks * 8 numbers, kThreads threads each (four rows to a block where a warp has a row).
//   kRing = false: a row a group of threads, loaded straight into registers: the shortest way for few rows, and for short ones.
//   kRing = true: groups walk over the rows, and copies bring the next ones into a ring in shared memory (P.slots rows), so that memory works while a row is reduced.
//   kExact: the row fills the threads' chunks, and nothing asks where it ends (8192 x 4096 through the norm 44.9 -> 41.4 us, into eight bits 18.9 -> 18.3).
// (Six blocks of the norm's 256 threads an SM: with five, which a few registers more make, 47.9 us.)
template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes, bool kRing, bool kExact>
__global__ void __launch_bounds__(kThreads == 32 ? 128 : kThreads, !kRing ? 0 : !kNorm || kThreads == 32 ? 1024 / (kThreads == 32 ? 128 : kThreads) : kChunks == 2 && kThreads <= 256 ? 1536 / kThreads : kThreads >= 512 ? 1024 / kThreads : 768 / kThreads) q8_rows_kernel(const Rows P) {
    constexpr int kWarps = kThreads / 32, kGroups = kThreads == 32 ? 4 : 1;
    constexpr bool kEarly = kNorm && !kRing && kChunks <= 2;       // the weight is asked for with the row, where registers allow
    // A slot is filled again when the row's threads have met for the first time where there may be but one slot a block (2000 x 16384 through the norm 42.5 us, 50.1 with one block an SM and three
    // slots; 2000 x 28672 of f32 into eight bits 50.1, 62.2 the other way), else when the row is done: thread 0's warp is then not held up in the row's chain (8192 x 14336 into eight bits 56.6 us, 61.2).
    constexpr bool kSoon = kThreads >= (kNorm ? 512 : 1024);
    constexpr uint32_t kXSize = kX32 ? 4 : 2, kRSize = kRes == kF32 ? 4 : kRes == kBf16 ? 2 : 0;
    __shared__ double sums[2][kWarps];
    __shared__ uint32_t tops[2][kWarps];
    __shared__ uint64_t full[kGroups][kMostSlots];
    __shared__ int abort_flag;
    extern __shared__ __align__(16) uint8_t ring[];
    const uint32_t t = threadIdx.x % kThreads, group = threadIdx.x / kThreads, warp = t >> 5;
    const uint64_t groups = (uint64_t)gridDim.x * kGroups, first = (uint64_t)blockIdx.x * kGroups + group;
    const uint32_t whole = P.dim & ~7u;                            // what the copies bring: whole chunks
    const uint32_t mine = ptx::smem_u32(ring) + group * P.slots * P.slot_bytes;
    ptx::grid_launch_dependents();
    if constexpr (kRing) {
        if (t == 0) {
            for (uint32_t s = 0; s < P.slots; ++s) ptx::mbar_init(ptx::smem_u32(&full[group][s]), 1);
            ptx::fence_barrier_init();
            ptx::fence_proxy_async_smem();
            abort_flag = 0;
        }
        __syncthreads();
    }
    ptx::grid_dependency_wait();
    const auto fill = [&](uint64_t row, uint32_t slot) {
        const uint32_t bar = ptx::smem_u32(&full[group][slot]), to = mine + slot * P.slot_bytes;
        ptx::mbar_arrive_expect_tx(bar, whole * (kXSize + kRSize));
        if (whole) ptx::bulk_load(to, (const char*)P.x + row * P.x_stride * kXSize, whole * kXSize, bar);
        if (kRes && whole) ptx::bulk_load(to + P.residual_at, (const char*)P.residual + row * P.residual_stride * kRSize, whole * kRSize, bar);
    };
    if constexpr (kRing) {
        if (t == 0)
            for (uint32_t s = 0; s < P.slots; ++s)
                if (first + s * groups < P.n_rows && !(P.drop_load && first + s * groups == 0)) fill(first + s * groups, s);     // (self-test of the failure path: row 0 is not brought)
    }
    uint32_t slot = 0, phase = 0, turn = 0;
    const auto refill = [&](uint64_t row) {
        if constexpr (kRing)
            if (t == 0 && row + P.slots * groups < P.n_rows) fill(row + P.slots * groups, slot);
    };
    uint64_t row = first;
    for (; row < P.n_rows; row += groups, turn ^= 1) {
        if constexpr (kRing) {
            if (!ptx::mbar_wait_warp(ptx::smem_u32(&full[group][slot]), phase, &abort_flag, P.wait_limit_ns)) {
                // The row's other warps may have had their answer before: they are told where they next meet, and all leave the loop at this row, with nothing of it written but what the sum is kept in.
                if ((t & 31) == 0) {
                    atomicCAS(P.status, 0, kStatusProducerTimeout | (int)(row & 0xFFFFFF));
                    if constexpr (kNorm) sums[turn][warp] = kGone;
                    else tops[turn][warp] = kGoneTop;
                }
                if constexpr (kWarps > 1) ptx::bar_sync(1, kThreads);
                break;
            }
        }
        const uint32_t in_ring = mine + slot * P.slot_bytes;
        const char* const x_row = (const char*)P.x + row * P.x_stride * kXSize;
        float2 v[kChunks][4], w[kEarly ? kChunks : 1][4];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const uint32_t e = (c * kThreads + t) * 8, have = kExact ? 8 : e < P.dim ? P.dim - e : 0;
            if (kRing && have >= 8) lds8<kX32>(v[c], in_ring + e * kXSize);
            else load8<kX32>(v[c], x_row, e, have);
            if constexpr (kEarly) {
                if (P.weight_f32) load8<true>(w[c], P.weight, e, have);
                else load8<false>(w[c], P.weight, e, have);
            }
        }
        if constexpr (kRes != kNone) {
            const char* const r_row = (const char*)P.residual + row * P.residual_stride * kRSize;
            char* const o_row = (char*)P.residual_out + row * P.residual_out_stride * kRSize;
            float2 u[kRing ? 1 : kChunks][4];                      // loads from memory are all asked for before one is waited for
            if constexpr (!kRing) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const uint32_t e = (c * kThreads + t) * 8;
                    load8<kRes == kF32>(u[c], r_row, e, kExact ? 8 : e < P.dim ? P.dim - e : 0);
                }
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8, have = kExact ? 8 : e < P.dim ? P.dim - e : 0;
                if constexpr (kRing) {
                    if (have >= 8) lds8<kRes == kF32>(u[0], in_ring + P.residual_at + e * kRSize);
                    else load8<kRes == kF32>(u[0], r_row, e, have);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[c][i] = add2(v[c][i], u[kRing ? 0 : c][i]);
                    if constexpr (kRes == kBf16) v[c][i] = unpack_bf16(pack_bf16(v[c][i]));
                }
                if (P.residual_out && have) store8<kRes == kF32>(o_row, e, have, v[c]);
            }
        }
        if constexpr (kNorm) {
            double part[4] = {0, 0, 0, 0};                         // squares of f32 are exact in f64
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const double a = v[c][i].x, b = v[c][i].y;
                    part[(i & 1) * 2] = fma(a, a, part[(i & 1) * 2]);
                    part[(i & 1) * 2 + 1] = fma(b, b, part[(i & 1) * 2 + 1]);
                }
            double sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
            if constexpr (kWarps > 1) {
                if ((t & 31) == 0) sums[turn][warp] = sum;
                ptx::bar_sync(1, kThreads);
                if constexpr (kSoon) refill(row);
                double s[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < kWarps; ++i) s[i & 3] += sums[turn][i];
                sum = (s[0] + s[1]) + (s[2] + s[3]);
            }
            const double mean = fma(sum, P.inv_dim, P.eps);
            if constexpr (kRing && kWarps > 1)
                if (!((float)mean > 1e-30f) && __any_sync(0xFFFFFFFFu, (t & 31) < kWarps && sums[turn][t & 31] == kGone)) break;
            const float r = (float)inverse_root(mean);
            const float2 r2 = make_float2(r, r);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8, have = kExact ? 8 : e < P.dim ? P.dim - e : 0;
                float2 f[4];
                if constexpr (!kEarly) {
                    if (P.weight_f32) load8<true>(f, P.weight, e, have);
                    else load8<false>(f, P.weight, e, have);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) v[c][i] = mul2(mul2(v[c][i], r2), kEarly ? w[c][i] : f[i]);
                if (have < 8) {                                    // what lies behind the row stays zero, whatever r is
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[c][i] = make_float2(2 * i < (int)have ? v[c][i].x : 0.0f, 2 * i + 1 < (int)have ? v[c][i].y : 0.0f);
                }
                if (P.y && have) store8<false>(P.y + row * P.y_stride, e, have, v[c]);
            }
        }
        if (!kNorm || P.q) {
            float most = 0;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = most_of(most, v[c][i]);
            // the bits of sizes are in their order, infinities and NaNs above all numbers
            uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most) & 0x7FFFFFFFu);
            if constexpr (kWarps > 1) {
                if ((t & 31) == 0) tops[turn][warp] = top;
                ptx::bar_sync(1, kThreads);
                if constexpr (kSoon && !kNorm) refill(row);
                top = 0;
#pragma unroll
                for (int i = 0; i < kWarps; ++i) top = max(top, tops[turn][i]);
                if (kRing && !kNorm && top == kGoneTop) break;
            }
            most = __uint_as_float(top);
            const bool held = most >= 0x1p-119f && top < 0x7F800000u;
            const float inverse = held ? __fdiv_rn(127.0f, most) : 0.0f;
            const float2 inverse2 = make_float2(inverse, inverse);
            if (t == 0) P.scales[row] = held ? __fdiv_rn(most, 127.0f) : top < 0x7F800000u ? 0.0f : __uint_as_float(0x7FFFFFFFu);
            int8_t* const q_row = P.q + row * P.q_stride;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8;
                if (!kExact && e >= P.dim) continue;
                uint2 b = make_uint2(bytes_of(mul2(v[c][0], inverse2), mul2(v[c][1], inverse2)), bytes_of(mul2(v[c][2], inverse2), mul2(v[c][3], inverse2)));
                if (!held) b = make_uint2(0, 0);                   // (products of infinities and NaNs)
                if (kExact || P.dim - e >= 8) {
                    *(uint2*)(q_row + e) = b;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < (int)(P.dim - e)) q_row[e + i] = (int8_t)((i < 4 ? b.x : b.y) >> (8 * (i & 3)));
                }
            }
        }
        if constexpr (kRing) {
            if constexpr (kWarps == 1) __syncwarp();               // (the others have met)
            if constexpr (!kSoon) refill(row);
            if (++slot == P.slots) slot = 0, phase ^= 1;
        } else {
            break;
        }
    }
    if constexpr (kRing) {
        // The rows were left: the copies that are on their way land before the block's shared memory is another's.  They are waited for again, a millisecond at most: the row's, those of the slots behind
        // it, and the slot's next one where it may have been asked for.
        if (row < P.n_rows && t == 0) {
            const uint64_t until = ptx::globaltimer_ns() + 1000000;
            for (uint32_t s = 0; s < P.slots + kSoon && row < P.n_rows; ++s, row += groups) {
                ptx::mbar_wait_until(ptx::smem_u32(&full[group][slot]), phase, until);
                if (++slot == P.slots) slot = 0, phase ^= 1;
            }
        }
    }
}

// A row a group of threads, straight into registers.
template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes>
cudaError_t launch_few(t0_runtime* rt, const Rows& P) {
    constexpr uint32_t kGroups = kThreads == 32 ? 4 : 1;
    return gemm::launch_pdl(q8_rows_kernel<kThreads, kChunks, kNorm, kX32, kRes, false, false>, (P.n_rows + kGroups - 1) / kGroups, kGroups * kThreads, 0, rt->stream, P);
}
// A row of x and one of the residual in the ring, each from a 128-byte boundary on.
template <bool kX32, int kRes>
void lay_out_slot(Rows& P) {
    P.residual_at = ((P.dim & ~7u) * (kX32 ? 4 : 2) + 127) & ~127u;
    P.slot_bytes = P.residual_at + (((P.dim & ~7u) * (kRes == kF32 ? 4 : kRes == kBf16 ? 2 : 0) + 127) & ~127u);
}
// (The caller has seen to it that one slot for each group is no more than kMostRing.)
template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes, bool kExact>
cudaError_t launch_ring(t0_runtime* rt, Rows& P) {
    constexpr uint32_t kGroups = kThreads == 32 ? 4 : 1, kRoom = 200u << 10, kAtOnce = std::max(1, (kNorm && kThreads < 512 ? 1536 : 1024) / (int)(kGroups * kThreads));
    lay_out_slot<kX32, kRes>(P);
    const uint32_t row_bytes = std::max(1u, kGroups * P.slot_bytes);
    const uint32_t at_once = std::max(1u, std::min(kAtOnce, kRoom / ((kNorm && kThreads >= 512 ? 1 : 2) * row_bytes)));       // blocks an SM
    P.slots = std::min(kMostSlots, std::max(1u, kRoom / at_once / row_bytes));
    P.drop_load = rt->drop_next_load.exchange(0) != 0;
    auto kern = q8_rows_kernel<kThreads, kChunks, kNorm, kX32, kRes, true, kExact>;
    static std::atomic<bool> ready[64];
    if (rt->device < 0 || rt->device >= 64) return cudaErrorInvalidDevice;
    if (!ready[rt->device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostRing);
        if (e != cudaSuccess) return e;
        ready[rt->device].store(true, std::memory_order_release);
    }
    const uint64_t blocks = ((uint64_t)P.n_rows + kGroups - 1) / kGroups;
    return gemm::launch_pdl(kern, (uint32_t)std::min<uint64_t>(blocks, (uint64_t)at_once * rt->sm_count), kGroups * kThreads, P.slots * row_bytes, rt->stream, P);
}

template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes>
cudaError_t launch_many(t0_runtime* rt, Rows& P) {
    if constexpr (kThreads > 32)
        if (P.dim == kThreads * kChunks * 8) return launch_ring<kThreads, kChunks, kNorm, kX32, kRes, true>(rt, P);
    return launch_ring<kThreads, kChunks, kNorm, kX32, kRes, false>(rt, P);
}

// As many rows as have a thread for each chunk of eight at the same time (2048 threads an SM): so many threads a row, for the shortest chain (one row of 4096 through the norm: 2.4 us; with 256
// threads and two chunks 2.9).  More rows: fewer threads each and the ring.  With the norm a row has a long chain of sums, which more threads shorten (8192 x 4096, 256 threads and two chunks /
// 128 and four / 64 and eight: 44.8 / 46.4 / 73.9 us); without it a thread's fixed work counts (8192 x 4096 with 256 / 128: 19.8 / 18.9; 16384 x 2048 with 128 / 64: 23.0 / 18.9).
// Short rows never take the ring, whose copies are too small to be worth their issue: up to 256 numbers a warp a row (30000 x 128 through the norm: 14.5 us, 25.2 with it), with the norm up to
// 1024 too (5000 x 1024: 10.3, 12.6 with it).
// Directly / with the ring, us: 600 x 4096 3.5 / 3.9, 1200 x 4096 5.0 / 4.6, 2500 x 1024 3.7 / 3.6, norm of 300 x 512 2.4 / 2.8, of 1200 x 512 4.1 / 3.8.
template <bool kNorm, bool kX32, int kRes>
cudaError_t launch_by_dim(t0_runtime* rt, Rows& P) {
    const uint32_t d = P.dim;
    if (d <= 256) return launch_few<32, 1, kNorm, kX32, kRes>(rt, P);
    const uint64_t threads = d <= 512 ? 64 : d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024;
    if (P.n_rows * threads <= 2048ull * rt->sm_count || (kNorm && d > 512 && d <= 1024))
        return d <= 512 ? launch_few<64, 1, kNorm, kX32, kRes>(rt, P) : d <= 1024 ? launch_few<128, 1, kNorm, kX32, kRes>(rt, P) : d <= 2048 ? launch_few<256, 1, kNorm, kX32, kRes>(rt, P)
             : d <= 4096 ? launch_few<512, 1, kNorm, kX32, kRes>(rt, P) : d <= 8192 ? launch_few<1024, 1, kNorm, kX32, kRes>(rt, P) : d <= 16384 ? launch_few<1024, 2, kNorm, kX32, kRes>(rt, P)
                         : launch_few<1024, 4, kNorm, kX32, kRes>(rt, P);
    if (d <= 512) return launch_many<32, 2, kNorm, kX32, kRes>(rt, P);
    if constexpr (!kNorm)
        if (d <= 1024) return launch_many<32, 4, kNorm, kX32, kRes>(rt, P);
    if constexpr (kNorm) {                                         // three chunks a thread where they are enough (4000 x 5120 42.7 -> 36.2 us, 2000 x 12288 42.6 -> 33.9)
        if (d > 4096 && d <= 6144) return launch_many<256, 3, kNorm, kX32, kRes>(rt, P);
        if (d > 8192 && d <= 12288) return launch_many<512, 3, kNorm, kX32, kRes>(rt, P);
    }
    if (d > 16384) {
        // rows of f32 with a residual of f32 from 28168 numbers on: one of each is longer than the ring can be, and every row goes straight into registers (1000 x 28672 82.0 us, 297 x 32768 37.1; with a ring
        // of one slot 1000 x 28160 takes 88.9)
        lay_out_slot<kX32, kRes>(P);
        return P.slot_bytes > kMostRing ? launch_few<1024, 4, kNorm, kX32, kRes>(rt, P) : launch_many<1024, 4, kNorm, kX32, kRes>(rt, P);
    }
    return d <= 2048 ? launch_many<kNorm ? 128 : 64, kNorm ? 2 : 4, kNorm, kX32, kRes>(rt, P) : d <= 4096 ? launch_many<kNorm ? 256 : 128, kNorm ? 2 : 4, kNorm, kX32, kRes>(rt, P)
         : d <= 8192 ? launch_many<256, 4, kNorm, kX32, kRes>(rt, P) : launch_many<512, 4, kNorm, kX32, kRes>(rt, P);
}

}  // namespace
}  // namespace q8
}  // namespace t0
