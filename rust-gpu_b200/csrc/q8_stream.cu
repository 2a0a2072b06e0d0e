// Products of few rows in eight bits, plain or gated: the weights are streamed once, tcgen05.mma kind::i8 with the WEIGHTS as its 128 rows and the tokens as its columns.
//
// What bounds these products is the weights' way from memory.  A tile is `rows` rows of the weights (up to 128, as many as give every SM the same share: the tensor core works on
// 128 whatever is in them) by `tokens` rows of A (a multiple of 16, up to 256; 128 for the gated pair, whose two matrices take a tile each), and a CTA takes a tile, or a part of its
// k blocks where the tiles of whole sums would be too few: the parts' CTAs form a cluster, park their sums in shared memory and share the adding out by tokens (whole numbers: the
// order is of no matter).  A lane of tensor memory is one row of the weights, so a store instruction writes 32 neighbouring numbers of one row of y whatever its alignment.
// 1 x 11008 x 4096 takes 10.0 us: 5.9 from the first block to the last (7.6 TB/s), the rest is launch (2.2), first operands (1.3) and epilogue (0.7).  Gated 100 x 14336 x 4096 takes 23.8: 15.8 for the
// blocks (7.4 TB/s), 2.2 until the first is there, 2.5 of epilogue.  Shared memory for 192 KB of stages, one CTA an SM: with 96 KB and two CTAs too little is on its way (10.6 and 19.0 us for one
// token plain and gated, 10.4 and 17.1 so).
#include "gemm_common.cuh"
#include "q8.cuh"
#include "runtime_internal.h"

namespace t0 {
namespace q8 {
namespace {

constexpr uint32_t kMostWarps = 2 + 16;             // producer, UMMA issuer, one to four epilogue warps for each quarter of the rows
constexpr uint32_t kBlock = 128;                     // codes a stage is deep
constexpr uint32_t kMaxStages = 32;
constexpr uint32_t kMostParts = 4;
constexpr uint32_t kTile = 128 * kBlock;             // bytes that the tensor core reads from where a tile of the weights begins, however many rows it has
constexpr uint32_t kMostRing = 192 * 1024;           // shared memory for stages
constexpr uint32_t kMostSmem = 1024 + kMostRing + kTile + 1024;

struct StreamParams {
    Product P;
    uint32_t rows, tokens;                           // of a tile
    uint32_t tiles_n, tiles_m, parts;
    uint32_t k_blocks, stages, ring;                 // the ring in bytes, with what the last tile is short of 128 rows
    uint32_t w_bytes, stage_bytes;                   // one matrix's rows of a stage (whole kilobytes), all of a stage
    uint32_t tmem_cols, drop_load;
    uint32_t ahead;                                  // blocks of a part that are asked into L2 before the launch waits for the one before it
    int* status;
    uint64_t wait_limit_ns;
};

// The rows of the weights from n0 on that are lanes of a warp, and what they are multiplied with.
struct Column {
    uint32_t n;
    bool in;
    float scale, scale2, bias;
};
template <bool kGated>
__device__ __forceinline__ Column column_of(const StreamParams& p, uint32_t n0, uint32_t lane_row) {
    Column c;
    c.n = n0 + lane_row;
    c.in = lane_row < p.rows && c.n < p.P.n;
    c.scale = c.in ? p.P.w_scales[0][c.n] : 0.0f;
    c.scale2 = kGated && c.in ? p.P.w_scales[1][c.n] : 0.0f;
    c.bias = !kGated && c.in && p.P.bias ? p.P.bias[c.n] : 0.0f;
    return c;
}
// kCount sums of this lane's column, of kCount tokens, to what y has there.
template <bool kGated, int kCount>
__device__ __forceinline__ void finish(const StreamParams& p, const Column& c, const int32_t (&sum)[kCount], const int32_t (&sum2)[kGated ? kCount : 1], const float (&a_scale)[kCount],
                                       float (&v)[kCount]) {
    const float2 w = make_float2(c.scale, c.scale), w2 = make_float2(c.scale2, c.scale2);
#pragma unroll
    for (int j = 0; j < kCount; j += 2) {
        const float2 x = scaled(sum[j], sum[j + 1], make_float2(a_scale[j], a_scale[j + 1]), w);
        v[j] = x.x, v[j + 1] = x.y;
    }
    if constexpr (kGated) {
        gate(v, p.P.act, p.P.out_bf16);
#pragma unroll
        for (int j = 0; j < kCount; j += 2) {
            const float2 x = mul2(make_float2(v[j], v[j + 1]), scaled(sum2[j], sum2[j + 1], make_float2(a_scale[j], a_scale[j + 1]), w2));
            v[j] = x.x, v[j + 1] = x.y;
        }
    } else if (p.P.bias) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) v[j] = __fadd_rn(v[j], c.bias);
    }
}
__device__ __forceinline__ void put(const StreamParams& p, const Column& c, uint64_t at, float v) {
    if (!c.in) return;
    if (p.P.out_bf16) ((__nv_bfloat16*)p.P.y)[at] = __float2bfloat16_rn(v);
    else ((float*)p.P.y)[at] = v;
}

// The parts' sums of this part's tokens, added and finished: a warp takes a quarter of the rows and every so many of the tokens, kAhead of them with the loads from all (up to kParts) parts in
// flight.  Scales are asked for before the parts meet.
template <bool kGated, uint32_t kParts, uint32_t kAhead>
__device__ __forceinline__ void add_parts(const StreamParams& p, uint32_t smem, uint32_t n0, uint32_t m0, uint32_t part, volatile int* abort_flag) {
    const Product& P = p.P;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tokens = min(p.tokens, P.m - m0), quarters = (min(p.rows, P.n - n0) + 31) / 32;
    const uint32_t quarter = warp % quarters, each = p.parts * ((blockDim.x / 32 - quarter + quarters - 1) / quarters);
    const Column c = column_of<kGated>(p, n0, quarter * 32 + lane);
    uint32_t t = part + warp / quarters * p.parts;
    float a_scale[kAhead];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j) a_scale[j] = t + j * each < tokens ? P.a_scales[m0 + t + j * each] : 0.0f;
    ptx::cluster_sync_all();
    if (*abort_flag) return;
    uint32_t from[kParts];
#pragma unroll
    for (uint32_t s = 0; s < kParts; ++s) from[s] = ptx::mapa(smem + (quarter * 32 + lane) * 4, min(s, p.parts - 1));
    while (t < tokens) {
        int32_t sum[kAhead], sum2[kGated ? kAhead : 1];
        {
            int32_t x[kParts][kAhead], x2[kGated ? kParts : 1][kAhead];
#pragma unroll
            for (uint32_t s = 0; s < kParts; ++s)
#pragma unroll
                for (uint32_t j = 0; j < kAhead; ++j) {
                    const uint32_t tt = min(t + j * each, tokens - 1);
                    x[s][j] = kParts == 2 || s < p.parts ? ptx::ld_cluster_i32(from[s] + tt * 512) : 0;
                    if constexpr (kGated) x2[s][j] = kParts == 2 || s < p.parts ? ptx::ld_cluster_i32(from[s] + (p.tokens + tt) * 512) : 0;
                }
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j) {
                sum[j] = x[0][j];
                if constexpr (kGated) sum2[j] = x2[0][j];
#pragma unroll
                for (uint32_t s = 1; s < kParts; ++s) {
                    sum[j] += x[s][j];
                    if constexpr (kGated) sum2[j] += x2[s][j];
                }
            }
        }
        float v[kAhead], next[kAhead];
        const uint32_t t1 = t + kAhead * each;
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) next[j] = t1 + j * each < tokens ? P.a_scales[m0 + t1 + j * each] : 0.0f;
        finish<kGated, kAhead>(p, c, sum, sum2, a_scale, v);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            if (t + j * each < tokens) put(p, c, (uint64_t)(m0 + t + j * each) * P.y_stride + c.n, v[j]);
            a_scale[j] = next[j];
        }
        t = t1;
    }
}

template <bool kGated>
__global__ void __launch_bounds__(32 * kMostWarps) q8_stream_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
                                                             const StreamParams p) {
    constexpr uint32_t kW = kGated ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + p.ring);
    uint64_t* full_bar = bars;
    uint64_t* empty_bar = bars + kMaxStages;
    uint64_t* done_bar = bars + 2 * kMaxStages;
    uint32_t* tmem_holder = (uint32_t*)(bars + 2 * kMaxStages + 1);
    volatile int* abort_flag = (volatile int*)(tmem_holder + 1);
    const Product& P = p.P;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t part = blockIdx.x % p.parts, tile = blockIdx.x / p.parts, n0 = tile / p.tiles_m * p.rows, m0 = tile % p.tiles_m * p.tokens;
    const uint32_t kb0 = (uint32_t)((uint64_t)p.k_blocks * part / p.parts), kb1 = (uint32_t)((uint64_t)p.k_blocks * (part + 1) / p.parts);
    // Every CTA begins at another block of its part: all read the same rows of A, and in step they would ask the same few lines of L2 at the same time.
    const uint32_t first = kb0 + (uint32_t)((uint64_t)tile * 2654435761ull % (kb1 - kb0));

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
        }
        ptx::mbar_init(ptx::smem_u32(done_bar), 1);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::tma_prefetch_desc(&map_a);
        ptx::tma_prefetch_desc(&map_w);
        if (kGated) ptx::tma_prefetch_desc(&map_w2);
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_holder), p.tmem_cols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_holder;
    ptx::grid_launch_dependents();
    if (warp == 0) {
        // What the launch before this one leaves idle of the memory's time: the first stages' weights on their way into L2 (a hint: whatever that launch still writes, L2 has it).
        const uint32_t issue = ptx::elect_one(), ahead = min(p.ahead, kb1 - kb0);
        for (uint32_t i = 0, kb = first; i < ahead; ++i, kb = kb + 1 == kb1 ? kb0 : kb + 1) {
            ptx::tma_prefetch_2d_if(issue, &map_w, (int32_t)(kb * kBlock), (int32_t)n0);
            if (kGated) ptx::tma_prefetch_2d_if(issue, &map_w2, (int32_t)(kb * kBlock), (int32_t)n0);
        }
    }
    ptx::grid_dependency_wait();

    if (warp == 0) {
        uint32_t stage = 0, phase = 0;
        for (uint32_t i = kb0, kb = first; i < kb1; ++i, kb = kb + 1 == kb1 ? kb0 : kb + 1) {
            if (!ptx::mbar_wait_warp(ptx::smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag, p.wait_limit_ns)) {
                if (lane == 0) atomicCAS(p.status, 0, kStatusProducerTimeout | (int)(tile & 0xFFFFFF));
                break;
            }
            const uint32_t issue = ptx::elect_one() && !(p.drop_load && blockIdx.x == 0 && i == 0);       // (self-test of the failure path)
            const uint32_t fb = ptx::smem_u32(&full_bar[stage]), to = ptx::smem_u32(smem) + stage * p.stage_bytes;
            ptx::mbar_arrive_expect_tx_if(issue, fb, (kW * p.rows + p.tokens) * kBlock);
            ptx::tma_load_2d_if(issue, to, &map_w, fb, (int32_t)(kb * kBlock), (int32_t)n0);
            if (kGated) ptx::tma_load_2d_if(issue, to + p.w_bytes, &map_w2, fb, (int32_t)(kb * kBlock), (int32_t)n0);
            ptx::tma_load_2d_if(issue, to + kW * p.w_bytes, &map_a, fb, (int32_t)(kb * kBlock), (int32_t)m0);
            if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
    } else if (warp == 1) {
        const uint32_t idesc = ptx::make_idesc_i8_s32(128, p.tokens);
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (uint32_t kb = kb0; kb < kb1; ++kb) {
            if (!ptx::mbar_wait_warp(ptx::smem_u32(&full_bar[stage]), phase, abort_flag, p.wait_limit_ns)) {
                if (lane == 0) atomicCAS(p.status, 0, kStatusMmaTimeout | (int)(tile & 0xFFFFFF));
                ok = false;
                break;
            }
            ptx::tc_fence_after_sync();
            const uint32_t issue = ptx::elect_one();
            const uint32_t w_lo = ptx::smem_desc_lo(ptx::smem_u32(smem) + stage * p.stage_bytes, 16), a_lo = w_lo + ((kW * p.w_bytes) >> 4);
#pragma unroll
            for (uint32_t e = 0; e < kBlock / 32; ++e) {
                ptx::umma_i8_ss_if(issue, tmem_base, w_lo + 2 * e, a_lo + 2 * e, idesc, kb != kb0 || e != 0 ? 1u : 0u);
                if (kGated) ptx::umma_i8_ss_if(issue, tmem_base + p.tokens, w_lo + (p.w_bytes >> 4) + 2 * e, a_lo + 2 * e, idesc, kb != kb0 || e != 0 ? 1u : 0u);
            }
            ptx::umma_commit_if(issue, ptx::smem_u32(&empty_bar[stage]));
            if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
        if (ok) ptx::umma_commit_if(ptx::elect_one(), ptx::smem_u32(done_bar));
    } else {
        const uint32_t quarter = warp & 3, turn = (warp - 2) >> 2, turns = (blockDim.x / 32 - 2) >> 2;
        const bool some = quarter * 32 < p.rows && n0 + quarter * 32 < P.n;          // of this warp's rows
        const uint32_t tokens = min(p.tokens, P.m - m0);
        const Column c = column_of<kGated>(p, n0, quarter * 32 + lane);
        // the scales of the tokens: this turn's are there before its sums are, the next one's asked for a turn ahead
        const auto scale_of = [&](uint32_t t) { return p.parts == 1 && t + (lane & 15) < tokens ? P.a_scales[m0 + t + (lane & 15)] : 0.0f; };
        float mine = scale_of(turn * 16);
        if (!ptx::mbar_wait_warp(ptx::smem_u32(done_bar), 0, abort_flag, p.wait_limit_ns)) {
            if (lane == 0) atomicCAS(p.status, 0, kStatusEpilogueTimeout | (int)(tile & 0xFFFFFF));
        } else if (some) {
            ptx::tc_fence_after_sync();
            const uint32_t tmem = tmem_base + ((quarter * 32) << 16);
            const uint32_t parked = ptx::smem_u32(smem) + (quarter * 32 + lane) * 4;
#pragma unroll 1
            for (uint32_t t = turn * 16; t < tokens; t += 16 * turns) {
                uint32_t r[16], r2[kGated ? 16 : 1];
                const float next = scale_of(t + 16 * turns);
                ptx::tmem_ld_32x32b_x16(tmem + t, r);
                if constexpr (kGated) ptx::tmem_ld_32x32b_x16(tmem + p.tokens + t, r2);
                ptx::tmem_ld_wait();
                if (p.parts == 1) {
                    float a_scale[16], v[16];
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) a_scale[j] = __shfl_sync(0xFFFFFFFFu, mine, j);
                    finish<kGated, 16>(p, c, (const int32_t(&)[16])r, (const int32_t(&)[kGated ? 16 : 1])r2, a_scale, v);
                    const uint64_t at = (uint64_t)(m0 + t) * P.y_stride + c.n;
                    if (t + 16 <= tokens) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j) put(p, c, at + j * P.y_stride, v[j]);
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j)
                            if (t + j < tokens) put(p, c, at + j * P.y_stride, v[j]);
                    }
                } else {
                    // over the ring, which is idle: all copies have landed and all products read them
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) {
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(parked + (t + j) * 512), "r"(r[j]) : "memory");
                        if constexpr (kGated) asm volatile("st.shared.b32 [%0], %1;" ::"r"(parked + (p.tokens + t + j) * 512), "r"(r2[j]) : "memory");
                    }
                }
                mine = next;
            }
        }
    }

    // ---------------------------------------------------------------- the parts' sums
    __syncwarp();
    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    ptx::tc_fence_before_sync();
    if (p.parts > 1) {
        // two tokens ahead (128 x 4096 x 4096 in four parts with one / two / four: 10.2 / 9.7 / 10.1 us; in two parts with two / four / eight: 9.2 / 9.4 / 9.3)
        if (p.parts == 2) add_parts<kGated, 2, 2>(p, ptx::smem_u32(smem), n0, m0, part, abort_flag);
        else add_parts<kGated, kMostParts, 2>(p, ptx::smem_u32(smem), n0, m0, part, abort_flag);
        ptx::cluster_sync_all();                       // a CTA's shared memory stays until all have read it
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, p.tmem_cols);
    }
}

template <bool kGated>
int launch_instance(t0_runtime* rt, const Product& P, const Cut& cut) {
    auto kern = q8_stream_kernel<kGated>;
    static std::atomic<bool> ready[64];
    const int dev = rt->device;
    if (dev < 0 || dev >= 64) return fail(T0_ERR_INVALID, "device ordinal out of range");
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostSmem);
        if (e != cudaSuccess) return fail(T0_ERR_CUDA, "cudaFuncSetAttribute(smem=%u): %s", kMostSmem, cudaGetErrorString(e));
        ready[dev].store(true, std::memory_order_release);
    }
    StreamParams p;
    memset((void*)&p, 0, sizeof p);
    p.P = P;
    p.rows = cut.rows; p.tokens = cut.tokens; p.parts = cut.parts;
    p.tiles_n = ceil_div(P.n, p.rows); p.tiles_m = ceil_div(P.m, p.tokens);
    p.k_blocks = ceil_div(P.k, kBlock);
    p.w_bytes = ((p.rows + 7) & ~7u) * kBlock;
    p.stage_bytes = (kGated ? 2 : 1) * p.w_bytes + p.tokens * kBlock;
    p.stages = std::min(kMaxStages, kMostRing / p.stage_bytes);
    p.ring = p.stages * p.stage_bytes + (p.w_bytes + p.tokens * kBlock < kTile ? kTile - p.w_bytes - p.tokens * kBlock : 0);
    if (p.parts > 1) p.ring = std::max(p.ring, (kGated ? 2 : 1) * p.tokens * 512);
    p.ahead = std::min(p.stages, 8u);
    p.tmem_cols = 32;
    while (p.tmem_cols < (kGated ? 2 : 1) * p.tokens) p.tmem_cols *= 2;
    p.status = rt->d_status;
    const uint64_t limit = rt->wait_limit_ns.load(std::memory_order_relaxed);
    p.wait_limit_ns = limit ? limit : ptx::kWaitLimitNs;
    p.drop_load = rt->drop_next_load.exchange(0) != 0;
    const uint64_t grid = (uint64_t)p.tiles_n * p.tiles_m * p.parts;
    if (grid > 0x7FFFFFFFull) return fail(T0_ERR_UNSUPPORTED, "m=%u, n=%u: too much for one launch", P.m, P.n);
    // epilogue warps: one to four turns of 16 tokens (1 x 11008 x 4096 with 4 / 8 / 16: 10.1 / 10.2 / 10.5 us; gated 100 x 14336 x 4096 with 8 / 16: 25.4 / 23.8)
    const uint32_t warps = p.tokens <= 16 ? 4 : p.tokens <= 64 ? 8 : 16;
    CUtensorMap ma, mw, mw2;
    int rc = make_map_codes(&ma, P.a, P.a_stride, P.m, P.k, p.tokens);
    if (rc == T0_OK) rc = make_map_codes(&mw, P.w[0], P.w_stride, P.n, P.k, p.rows);
    mw2 = mw;
    if (rc == T0_OK && kGated) rc = make_map_codes(&mw2, P.w[1], P.w_stride, P.n, P.k, p.rows);
    if (rc != T0_OK) return rc;
    const cudaError_t e = gemm::launch_pdl_clusters(kern, (uint32_t)grid, p.parts, 32 * (2 + warps), 1024 + p.ring + 1024, rt->stream, ma, mw, mw2, p);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the eight-bit product failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

}  // namespace

int launch_stream(t0_runtime* rt, const Product& P, bool gated, const Cut& cut) {
    const DeviceGuard guard(rt->device);
    return gated ? launch_instance<true>(rt, P, cut) : launch_instance<false>(rt, P, cut);
}

}  // namespace q8
}  // namespace t0
