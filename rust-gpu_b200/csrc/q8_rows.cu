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

constexpr uint32_t kMostSlots = 16;

struct Rows {
    const void *x, *residual, *weight;
    void* residual_out;
    int8_t* q;
    float* scales;
    __nv_bfloat16* y;
    uint64_t x_stride, residual_stride, residual_out_stride, q_stride, y_stride;
    uint32_t n_rows, dim;
    uint32_t slots, slot_bytes, residual_at;           // the ring: rows, bytes a row, where in it the residual begins
    int* status;
    uint64_t wait_limit_ns;
    double inv_dim, eps;
    bool x_f32, residual_f32, weight_f32;
};

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

// Rows of up to kThreads * kChunks * 8 numbers, kThreads threads each (four rows to a block where a warp has a row).
//   kRing = false: a row a group of threads, loaded straight into registers: the shortest way for few rows, and for short ones.
//   kRing = true: groups walk over the rows, and copies bring the next ones into a ring in shared memory (P.slots rows), so that memory works while a row is reduced; a slot is filled again
//     as soon as all threads have taken its numbers into registers.
template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes, bool kRing>
__global__ void __launch_bounds__(kThreads == 32 ? 128 : kThreads) q8_rows_kernel(const Rows P) {
    constexpr int kWarps = kThreads / 32, kGroups = kThreads == 32 ? 4 : 1;
    constexpr bool kEarly = kNorm && !kRing && kChunks <= 2;       // the weight is asked for with the row, where registers allow
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
                if (first + s * groups < P.n_rows) fill(first + s * groups, s);
    }
    uint32_t slot = 0, phase = 0, turn = 0;
    for (uint64_t row = first; row < P.n_rows; row += groups, turn ^= 1) {
        if constexpr (kRing) {
            if (!ptx::mbar_wait_warp(ptx::smem_u32(&full[group][slot]), phase, &abort_flag, P.wait_limit_ns) && (t & 31) == 0) atomicCAS(P.status, 0, kStatusProducerTimeout | (int)(row & 0xFFFFFF));
        }
        const uint32_t in_ring = mine + slot * P.slot_bytes;
        const char* const x_row = (const char*)P.x + row * P.x_stride * kXSize;
        float2 v[kChunks][4], w[kEarly ? kChunks : 1][4];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const uint32_t e = (c * kThreads + t) * 8, have = e < P.dim ? P.dim - e : 0;
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
                    load8<kRes == kF32>(u[c], r_row, e, e < P.dim ? P.dim - e : 0);
                }
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8, have = e < P.dim ? P.dim - e : 0;
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
                __syncthreads();
                double s[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < kWarps; ++i) s[i & 3] += sums[turn][i];
                sum = (s[0] + s[1]) + (s[2] + s[3]);
            }
            const float r = (float)inverse_root(fma(sum, P.inv_dim, P.eps));
            const float2 r2 = make_float2(r, r);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t e = (c * kThreads + t) * 8, have = e < P.dim ? P.dim - e : 0;
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
                __syncthreads();
                top = 0;
#pragma unroll
                for (int i = 0; i < kWarps; ++i) top = max(top, tops[turn][i]);
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
                if (e >= P.dim) continue;
                uint2 b = make_uint2(bytes_of(mul2(v[c][0], inverse2), mul2(v[c][1], inverse2)), bytes_of(mul2(v[c][2], inverse2), mul2(v[c][3], inverse2)));
                if (!held) b = make_uint2(0, 0);                   // (products of infinities and NaNs)
                if (P.dim - e >= 8) {
                    *(uint2*)(q_row + e) = b;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < (int)(P.dim - e)) q_row[e + i] = (int8_t)((i < 4 ? b.x : b.y) >> (8 * (i & 3)));
                }
            }
        }
        if constexpr (kRing) {
            // all threads have met since they took the slot's numbers (a warp that has a row to itself meets here)
            if constexpr (kWarps == 1) __syncwarp();
            if (t == 0 && row + P.slots * groups < P.n_rows) fill(row + P.slots * groups, slot);
            if (++slot == P.slots) slot = 0, phase ^= 1;
        } else {
            break;
        }
    }
    if constexpr (kRing) {
        if (*(volatile int*)&abort_flag)                           // copies that were given up on may still be on their way
            for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
}

// A row a group of threads, straight into registers.
template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes>
cudaError_t launch_few(t0_runtime* rt, const Rows& P) {
    constexpr uint32_t kGroups = kThreads == 32 ? 4 : 1;
    return gemm::launch_pdl(q8_rows_kernel<kThreads, kChunks, kNorm, kX32, kRes, false>, (P.n_rows + kGroups - 1) / kGroups, kGroups * kThreads, 0, rt->stream, P);
}
template <int kThreads, int kChunks, bool kNorm, bool kX32, int kRes>
cudaError_t launch_many(t0_runtime* rt, Rows& P) {
    constexpr uint32_t kGroups = kThreads == 32 ? 4 : 1, kRoom = 200u << 10, kAtOnce = std::max(1, (kNorm ? 1536 : 1024) / (int)(kGroups * kThreads));
    P.residual_at = ((P.dim & ~7u) * (kX32 ? 4 : 2) + 127) & ~127u;
    P.slot_bytes = P.residual_at + (((P.dim & ~7u) * (kRes == kF32 ? 4 : kRes == kBf16 ? 2 : 0) + 127) & ~127u);
    const uint32_t row_bytes = std::max(1u, kGroups * P.slot_bytes);
    const uint32_t at_once = std::max(1u, std::min(kAtOnce, kRoom / (2 * row_bytes)));       // blocks an SM
    P.slots = std::min(kMostSlots, std::max(1u, kRoom / at_once / row_bytes));
    auto kern = q8_rows_kernel<kThreads, kChunks, kNorm, kX32, kRes, true>;
    static std::atomic<bool> ready[64];
    if (rt->device < 0 || rt->device >= 64) return cudaErrorInvalidDevice;
    if (!ready[rt->device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 << 10);
        if (e != cudaSuccess) return e;
        ready[rt->device].store(true, std::memory_order_release);
    }
    const uint64_t blocks = ((uint64_t)P.n_rows + kGroups - 1) / kGroups;
    return gemm::launch_pdl(kern, (uint32_t)std::min<uint64_t>(blocks, (uint64_t)at_once * rt->sm_count), kGroups * kThreads, P.slots * row_bytes, rt->stream, P);
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
    return d <= 2048 ? launch_many<kNorm ? 128 : 64, kNorm ? 2 : 4, kNorm, kX32, kRes>(rt, P) : d <= 4096 ? launch_many<kNorm ? 256 : 128, kNorm ? 2 : 4, kNorm, kX32, kRes>(rt, P)
         : d <= 8192 ? launch_many<256, 4, kNorm, kX32, kRes>(rt, P) : d <= 16384 ? launch_many<kNorm ? 1024 : 512, kNorm ? 2 : 4, kNorm, kX32, kRes>(rt, P)
                     : launch_many<1024, 4, kNorm, kX32, kRes>(rt, P);
}

template <bool kNorm>
int launch_rows(t0_runtime* rt, Rows& P) {
    const DeviceGuard guard(rt->device);
    P.status = rt->d_status;
    const uint64_t limit = rt->wait_limit_ns.load(std::memory_order_relaxed);
    P.wait_limit_ns = limit ? limit : ptx::kWaitLimitNs;
    cudaError_t e;
    if constexpr (kNorm) {
        const int res = !P.residual ? kNone : P.residual_f32 ? kF32 : kBf16;
        e = P.x_f32 ? (res == kNone ? launch_by_dim<true, true, kNone>(rt, P) : res == kF32 ? launch_by_dim<true, true, kF32>(rt, P) : launch_by_dim<true, true, kBf16>(rt, P))
                    : (res == kNone ? launch_by_dim<true, false, kNone>(rt, P) : res == kF32 ? launch_by_dim<true, false, kF32>(rt, P) : launch_by_dim<true, false, kBf16>(rt, P));
    } else {
        e = P.x_f32 ? launch_by_dim<false, true, kNone>(rt, P) : launch_by_dim<false, false, kNone>(rt, P);
    }
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the rows in eight bits failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

struct Back {
    const int8_t* q;
    const float* scales;
    void* y;
    uint64_t q_stride, y_stride;
    uint64_t chunks;                                   // of all rows
    uint32_t dim, per_row, magic;                      // chunks a row; 2^32 / per_row, rounded up
};

// Eight codes a chunk, so that a warp's stores stand side by side, and four chunks a thread, asked for together: 1024 chunks a block, whatever rows they are of.
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
    memset(&P, 0, sizeof P);
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
