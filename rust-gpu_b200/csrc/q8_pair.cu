// Products of many rows in eight bits, plain or gated, on CTA pairs: tcgen05.mma kind::i8 (cta_group::2), exact i32 sums in tensor memory, scales, bias and gate in the epilogue.
//
// A pair shares a 256 x 256 tile of sums: each CTA holds its 128 rows of A and half of the 256 rows of B, 128 codes deep a stage (16 KiB each, six stages).  A stage is 512 clocks of
// the tensor pipe, as a stage of 64 bf16 is, and moves as many bytes: the roles are those of the bf16 pair kernel, and so is the order of the tiles.
// The gated pair of products takes 128 rows of each matrix as the two halves of B: the even CTA loads the gate's, the odd one the other's, and the sums of one output stand in one
// lane of tensor memory, 128 columns apart.  The tile gives 256 x 128 outputs, and neither product leaves the SM.
// A last round that would leave half of the pairs idle is taken in half tiles.
// 8192 x 14336 x 4096 takes 300 to 347 us by how warm the GPU is (2.8 to 3.2 POP/s, twice its bf16 rate), the gated pair 4096 x 11008 x 4096 236 to 258: the tensor pipe is busy 89 to 91 % of
// the time and the power limit sets its clock.  Tiles of half the columns are bound by their operands' way from L2 (24 KB a block and CTA at 104 bytes a nanosecond): 256 x 4096 x 4096 12.8 us.
#include "gemm_common.cuh"
#include "q8.cuh"
#include "runtime_internal.h"

namespace t0 {
namespace q8 {

int make_map_codes(CUtensorMap* map, const int8_t* codes, uint64_t stride, uint32_t rows, uint32_t length, uint32_t box_rows) {
    gemm::EncodeTiledFn enc = gemm::get_encode_fn();
    if (!enc) return fail(T0_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {length, rows};
    cuuint64_t strides[1] = {stride};
    cuuint32_t box[2] = {128, box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(T0_ERR_CUDA, "cuTensorMapEncodeTiled (codes, %u x %u) failed: %d", rows, length, (int)r);
    return T0_OK;
}

namespace {

constexpr uint32_t kEpilogueWarps = 8, kThreads = 64 + 32 * kEpilogueWarps;   // producer, UMMA issuer, two epilogue warps for each quarter of the rows
constexpr uint32_t kHalf = 128;                      // rows of A, and of B, that one CTA loads
constexpr uint32_t kBlock = 128;                     // codes a stage is deep
constexpr uint32_t kOperandBytes = kHalf * kBlock, kStageBytes = 2 * kOperandBytes;
constexpr uint32_t kStages = 6;
constexpr uint32_t kRaster = 8;                      // column tiles that are walked together, so that their B stays in L2

struct PairParams {
    Product P;
    uint32_t tiles_m, tiles_n, k_blocks;
    uint32_t whole;                                  // tiles that are taken whole; those after them are taken in two halves of their columns
    uint32_t tma_store, drop_load;
    int* status;
    uint64_t wait_limit_ns;
};

struct Tile { uint32_t m, n, half; bool halved; };
__device__ __forceinline__ Tile tile_of(uint32_t i, const PairParams& p) {
    const bool halved = i >= p.whole;
    const uint32_t w = halved ? p.whole + (i - p.whole) / 2 : i, half = halved ? (i - p.whole) & 1u : 0u;
    const uint32_t group = w / (kRaster * p.tiles_m), first = group * kRaster, wide = min(kRaster, p.tiles_n - first), r = w - group * kRaster * p.tiles_m;
    return {r / wide, first + r % wide, half, halved};
}

constexpr uint32_t smem_bytes() { return kStages * kStageBytes + kEpilogueWarps * (gemm::kEpiStageBytes + 256) + 256; }

__device__ __forceinline__ uint32_t lds_word(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// 32 rows x 32 columns on their way to y, this lane's row `row0 + lane`: through `stage` (a 4 KiB block of this warp, 16-byte slots turned by the row) and out as one tiled TMA
// store a block (f32: a chunk; bf16: the two chunks of 64 columns, `half` of it) where y's rows begin and end on 16-byte boundaries, else row by row.
__device__ __forceinline__ void put_chunk(const PairParams& p, const CUtensorMap* map_y, const float (&v)[32], uint32_t row0, uint32_t col0, uint32_t which, uint32_t lane, uint32_t stage) {
    const Product& P = p.P;
    if (p.tma_store && (!P.out_bf16 || which == 0)) {
        if (lane == 0) ptx::bulk_wait_group_read_all();        // the block's last store has read it
        __syncwarp();
    }
    if (P.out_bf16) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            uint32_t q[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]);
                q[i] = *(const uint32_t*)&h;
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + (lane * 8 + ((which * 4 + j) ^ (lane & 7))) * 16), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]) : "memory");
        }
        if (which == 0 && col0 + 32 < P.n) return;             // the second chunk completes the block
        col0 -= which * 32;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(stage + (lane * 8 + (j ^ (lane & 7))) * 16), "f"(v[4 * j]), "f"(v[4 * j + 1]), "f"(v[4 * j + 2]), "f"(v[4 * j + 3]) : "memory");
    }
    if (p.tma_store) {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            ptx::tma_store_2d(map_y, stage, (int32_t)col0, (int32_t)row0);
            ptx::bulk_commit_group();
        }
        return;
    }
    __syncwarp();
    // 32-bit words wherever the row begins: a bf16 row at an odd number is written from its second number on, its first and last alone.  (Stores of two bytes a lane left twice as many
    // 32-byte sectors part written: 6959 x 1165 x 1684 took 32.3 us with them, 22.6 with these; n = 1168, with TMA stores, takes 15.7.)
    const uint32_t rows = min(32u, P.m - row0), cols = min(P.out_bf16 ? 64u : 32u, P.n - col0), slot = lane >> 2, in = stage + (lane & 3) * 4;
    const uint64_t step = P.y_stride * (P.out_bf16 ? 2 : 4);
    char* y = (char*)P.y + row0 * step + col0 * (P.out_bf16 ? 2 : 4);
    if (!P.out_bf16) {
        y += 4 * lane;
        if (rows == 32 && cols == 32) {
#pragma unroll
            for (uint32_t r = 0; r < 32; ++r, y += step) *(uint32_t*)y = lds_word(in + r * 128 + ((slot ^ (r & 7)) << 4));
        } else {
#pragma unroll 4
            for (uint32_t r = 0; r < rows; ++r, y += step) {
                const uint32_t q = lds_word(in + r * 128 + ((slot ^ (r & 7)) << 4));
                if (lane < cols) *(uint32_t*)y = q;
            }
        }
    } else {
#pragma unroll 8
        for (uint32_t r = 0; r < rows; ++r, y += step) {
            const uint32_t q = lds_word(in + r * 128 + ((slot ^ (r & 7)) << 4));
            uint16_t* const at = (uint16_t*)y + 2 * lane;
            if (((uintptr_t)y & 2) == 0) {
                if (2 * lane + 1 < cols) *(uint32_t*)at = q;
                else if (2 * lane < cols) *at = (uint16_t)q;
            } else {
                const uint32_t next = __shfl_down_sync(0xFFFFFFFFu, q, 1);
                if (lane == 0) *at = (uint16_t)q;
                if (2 * lane + 2 < cols) *(uint32_t*)(at + 1) = __byte_perm(q, next, 0x5432);
                else if (2 * lane + 1 < cols) at[1] = (uint16_t)(q >> 16);
            }
        }
    }
    __syncwarp();
}

// Scales (or biases) of 32 columns, one a lane, to all lanes: through 128 bytes of shared memory.
__device__ __forceinline__ void spread(uint32_t at, float mine, uint32_t lane) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + lane * 4), "f"(mine) : "memory"); }
__device__ __forceinline__ float4 spread4(uint32_t at, uint32_t j) {
    float4 f;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at + j * 16) : "memory");
    return f;
}

template <bool kGated>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
q8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w2,
               const __grid_constant__ CUtensorMap map_w_half, const __grid_constant__ CUtensorMap map_w2_half, const __grid_constant__ CUtensorMap map_y,
               const PairParams p) {
    constexpr uint32_t kWide = kGated ? 128 : 256;               // columns of y a tile has
    constexpr uint32_t kIdesc = ptx::make_idesc_i8_s32(256, 256), kIdescHalf = ptx::make_idesc_i8_s32(256, 128);
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* a_tiles = smem;
    uint8_t* b_tiles = smem + kStages * kOperandBytes;
    uint8_t* epi_stage = smem + kStages * kStageBytes;           // a block for each epilogue warp
    uint8_t* epi_cols = epi_stage + kEpilogueWarps * gemm::kEpiStageBytes;       // 2 x 32 numbers likewise
    uint64_t* bars = (uint64_t*)(epi_cols + kEpilogueWarps * 256);
    uint64_t* full_bar = bars;                                   // used in the even CTA only
    uint64_t* empty_bar = bars + kStages;
    uint64_t* tmem_full_bar = bars + 2 * kStages;
    uint64_t* tmem_empty_bar = bars + 2 * kStages + 2;           // used in the even CTA only
    uint32_t* tmem_holder = (uint32_t*)(bars + 2 * kStages + 4);
    volatile int* abort_flag = (volatile int*)(tmem_holder + 1);
    const Product& P = p.P;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta_rank = ptx::cluster_ctarank(), pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t total = p.whole + 2 * (p.tiles_m * p.tiles_n - p.whole);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            ptx::mbar_init(ptx::smem_u32(&tmem_full_bar[b]), 1);
            ptx::mbar_init(ptx::smem_u32(&tmem_empty_bar[b]), 2 * kEpilogueWarps);
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::tma_prefetch_desc(&map_a);
        ptx::tma_prefetch_desc(cta_rank ? &map_w2 : &map_w);
        if (p.tma_store) ptx::tma_prefetch_desc(&map_y);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_holder), 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_holder;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();

    if (warp == 0) {
        // ------------------------------------------------------------ copies (both CTAs): this CTA's rows of A, its half of B
        const CUtensorMap* const my_w = kGated && cta_rank ? &map_w2 : &map_w;
        const CUtensorMap* const my_w_half = kGated && cta_rank ? &map_w2_half : &map_w_half;
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (uint32_t w = pair_id; ok && w < total; w += n_pairs) {
            const Tile t = tile_of(w, p);
            const int32_t row = (int32_t)(t.m * 256 + cta_rank * kHalf), col = (int32_t)(t.n * kWide + t.half * (kWide / 2) + (kGated ? 0 : cta_rank * (t.halved ? kHalf / 2 : kHalf)));
            for (uint32_t kb = 0; kb < p.k_blocks; ++kb) {
                if (!ptx::mbar_wait_warp(ptx::smem_u32(&empty_bar[stage]), phase ^ 1, abort_flag, p.wait_limit_ns)) {
                    if (lane == 0) atomicCAS(p.status, 0, kStatusProducerTimeout | (int)(w & 0xFFFFFF));
                    ok = false;
                    break;
                }
                if (!(p.drop_load && pair_id == 0 && w == 0 && kb == 0) && ptx::elect_one()) {    // (self-test of the failure path: neither CTA of pair 0 fills its first stage)
                    const uint32_t fb_local = ptx::smem_u32(&full_bar[stage]);
                    if (cta_rank == 0) ptx::mbar_arrive_expect_tx(fb_local, t.halved ? 2 * (kOperandBytes + kOperandBytes / 2) : 2 * kStageBytes);
                    const uint32_t fb = ptx::mapa(fb_local, 0);
                    ptx::tma_load_2d_pair(ptx::smem_u32(a_tiles + stage * kOperandBytes), &map_a, fb, (int32_t)(kb * kBlock), row);
                    ptx::tma_load_2d_pair(ptx::smem_u32(b_tiles + stage * kOperandBytes), t.halved ? my_w_half : my_w, fb, (int32_t)(kb * kBlock), col);
                }
                __syncwarp();
                if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ products (even CTA)
        if (cta_rank == 0) {
            uint32_t stage = 0, phase = 0, iter = 0;
            bool ok = true;
            for (uint32_t w = pair_id; ok && w < total; w += n_pairs, ++iter) {
                const uint32_t buf = iter & 1, acc_phase = (iter >> 1) & 1;
                if (!ptx::mbar_wait_warp(ptx::smem_u32(&tmem_empty_bar[buf]), acc_phase ^ 1, abort_flag, p.wait_limit_ns)) {
                    if (lane == 0) atomicCAS(p.status, 0, kStatusMmaTimeout | (int)(w & 0xFFFFFF));
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t tmem_d = tmem_base + buf * 256, idesc = w >= p.whole ? kIdescHalf : kIdesc;
                for (uint32_t kb = 0; kb < p.k_blocks; ++kb) {
                    if (!ptx::mbar_wait_warp(ptx::smem_u32(&full_bar[stage]), phase, abort_flag, p.wait_limit_ns)) {
                        if (lane == 0) atomicCAS(p.status, 0, kStatusMmaTimeout | 0x800000 | (int)(w & 0x7FFFFF));
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    if (ptx::elect_one()) {
                        const uint32_t a_addr = ptx::smem_u32(a_tiles + stage * kOperandBytes), b_addr = ptx::smem_u32(b_tiles + stage * kOperandBytes);
#pragma unroll
                        for (uint32_t e = 0; e < kBlock / 32; ++e)
                            ptx::umma_i8_ss_pair(tmem_d, ptx::make_smem_desc(a_addr + e * 32, 16, 1024), ptx::make_smem_desc(b_addr + e * 32, 16, 1024), idesc, kb != 0 || e != 0 ? 1u : 0u);
                        const uint32_t eb = ptx::smem_u32(&empty_bar[stage]);
                        ptx::umma_commit_pair(eb);
                        ptx::umma_commit_pair(ptx::mapa(eb, 1));
                    }
                    __syncwarp();
                    if (++stage == kStages) { stage = 0; phase ^= 1; }
                }
                if (ok && ptx::elect_one()) {
                    const uint32_t tb = ptx::smem_u32(&tmem_full_bar[buf]);
                    ptx::umma_commit_pair(tb);
                    ptx::umma_commit_pair(ptx::mapa(tb, 1));
                }
                __syncwarp();
            }
        }
    } else {
        // ------------------------------------------------------------ sums to y (both CTAs): a quarter's two warps take its columns in turns of 64
        const uint32_t quarter = warp & 3, turn = (warp - 2) >> 2, stage = ptx::smem_u32(epi_stage) + (warp - 2) * gemm::kEpiStageBytes, cols = ptx::smem_u32(epi_cols) + (warp - 2) * 256;
        uint32_t iter = 0;
        for (uint32_t w = pair_id; w < total; w += n_pairs, ++iter) {
            const Tile t = tile_of(w, p);
            const uint32_t buf = iter & 1, acc_phase = (iter >> 1) & 1;
            const uint32_t row0 = t.m * 256 + cta_rank * kHalf + quarter * 32, row = row0 + lane;
            const float a_scale = row < P.m ? P.a_scales[row] : 0.0f;
            __syncwarp();
            if (!ptx::mbar_wait_warp(ptx::smem_u32(&tmem_full_bar[buf]), acc_phase, abort_flag, p.wait_limit_ns)) {
                if (lane == 0) atomicCAS(p.status, 0, kStatusEpilogueTimeout | (int)(w & 0xFFFFFF));
                break;
            }
            ptx::tc_fence_after_sync();
            const uint32_t tmem = tmem_base + ((quarter * 32) << 16) + buf * 256, wide = t.halved ? kWide / 2 : kWide;
#pragma unroll 1
            for (uint32_t i = 0;; ++i) {
                const uint32_t c = (i >> 1) * 4 + turn * 2 + (i & 1);
                if (c * 32 >= wide) break;
                const uint32_t col0 = t.n * kWide + t.half * (kWide / 2) + c * 32;
                if (col0 >= P.n || row0 >= P.m) break;
                const bool in = col0 + lane < P.n;
                spread(cols, in ? P.w_scales[0][col0 + lane] : 0.0f, lane);
                if (kGated) spread(cols + 128, in ? P.w_scales[1][col0 + lane] : 0.0f, lane);
                else if (P.bias) spread(cols + 128, in ? P.bias[col0 + lane] : 0.0f, lane);
                uint32_t r[32], r2[kGated ? 32 : 1];
                ptx::tmem_ld_32x32b_x32(tmem + c * 32, r);
                if constexpr (kGated) ptx::tmem_ld_32x32b_x32(tmem + wide + c * 32, r2);
                ptx::tmem_ld_wait();
                __syncwarp();
                float v[32];
                const float2 a2 = make_float2(a_scale, a_scale);
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const float4 s = spread4(cols, j);
                    const float2 x = scaled((int)r[4 * j], (int)r[4 * j + 1], a2, make_float2(s.x, s.y)), y = scaled((int)r[4 * j + 2], (int)r[4 * j + 3], a2, make_float2(s.z, s.w));
                    v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = y.x, v[4 * j + 3] = y.y;
                }
                if constexpr (kGated) {
                    gate(v, P.act, P.out_bf16);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const float4 s = spread4(cols + 128, j);
                        const float2 x = mul2(make_float2(v[4 * j], v[4 * j + 1]), scaled((int)r2[4 * j], (int)r2[4 * j + 1], a2, make_float2(s.x, s.y)));
                        const float2 y = mul2(make_float2(v[4 * j + 2], v[4 * j + 3]), scaled((int)r2[4 * j + 2], (int)r2[4 * j + 3], a2, make_float2(s.z, s.w)));
                        v[4 * j] = x.x, v[4 * j + 1] = x.y, v[4 * j + 2] = y.x, v[4 * j + 3] = y.y;
                    }
                } else if (P.bias) {
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const float4 s = spread4(cols + 128, j);
                        v[4 * j] = __fadd_rn(v[4 * j], s.x); v[4 * j + 1] = __fadd_rn(v[4 * j + 1], s.y); v[4 * j + 2] = __fadd_rn(v[4 * j + 2], s.z); v[4 * j + 3] = __fadd_rn(v[4 * j + 3], s.w);
                    }
                }
                put_chunk(p, &map_y, v, row0, col0, c & 1, lane, stage);
                __syncwarp();                                    // the next chunk's numbers take the place of this one's
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                const uint32_t te = ptx::smem_u32(&tmem_empty_bar[buf]);
                if (cta_rank == 0) ptx::mbar_arrive(te);
                else ptx::mbar_arrive_cluster(ptx::mapa(te, 0));
            }
        }
        if (p.tma_store && lane == 0) ptx::bulk_wait_group_all();
    }

    // ---------------------------------------------------------------- common exit
    __syncwarp();
    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

// y as the epilogue's TMA stores see it: boxes of 32 rows x 128 bytes.
int make_map_y(CUtensorMap* map, const Product& P) {
    gemm::EncodeTiledFn enc = gemm::get_encode_fn();
    if (!enc) return fail(T0_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const uint32_t size = P.out_bf16 ? 2 : 4;
    cuuint64_t dims[2] = {P.n, P.m};
    cuuint64_t strides[1] = {P.y_stride * size};
    cuuint32_t box[2] = {128 / size, 32};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, P.out_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, P.y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(T0_ERR_CUDA, "cuTensorMapEncodeTiled (y, %u x %u) failed: %d", P.m, P.n, (int)r);
    return T0_OK;
}

template <bool kGated>
int launch_instance(t0_runtime* rt, const Product& P) {
    auto kern = q8_pair_kernel<kGated>;
    static std::atomic<int> max_pairs[64];
    const int dev = rt->device;
    if (dev < 0 || dev >= 64) return fail(T0_ERR_INVALID, "device ordinal out of range");
    int pairs = max_pairs[dev].load(std::memory_order_acquire);
    if (pairs == 0) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes());
        if (e != cudaSuccess) return fail(T0_ERR_CUDA, "cudaFuncSetAttribute(smem=%u): %s", smem_bytes(), cudaGetErrorString(e));
        cudaLaunchConfig_t qc = {};
        qc.gridDim = dim3(2 * ((uint32_t)rt->sm_count / 2), 1, 1);
        qc.blockDim = dim3(kThreads, 1, 1);
        qc.dynamicSmemBytes = smem_bytes();
        e = cudaOccupancyMaxActiveClusters(&pairs, kern, &qc);
        if (e != cudaSuccess || pairs <= 0) { cudaGetLastError(); pairs = rt->sm_count / 2; }
        max_pairs[dev].store(pairs, std::memory_order_release);
    }
    PairParams p;
    memset((void*)&p, 0, sizeof p);
    p.P = P;
    p.tiles_m = ceil_div(P.m, 256);
    p.tiles_n = ceil_div(P.n, kGated ? 128 : 256);
    p.k_blocks = ceil_div(P.k, kBlock);
    const uint64_t total = (uint64_t)p.tiles_m * p.tiles_n;
    if (total > 0x7FFFFFFFull / kRaster) return fail(T0_ERR_UNSUPPORTED, "m=%u, n=%u: too much for one launch", P.m, P.n);
    // the last round of tiles, where it would leave half of the pairs idle or more: in halves, on twice as many
    const uint32_t rest = (uint32_t)(total % (uint64_t)pairs);
    p.whole = (uint32_t)total - (2 * rest <= (uint32_t)pairs ? rest : 0);
    const uint64_t items = p.whole + 2 * (total - p.whole);
    p.status = rt->d_status;
    const uint64_t limit = rt->wait_limit_ns.load(std::memory_order_relaxed);
    p.wait_limit_ns = limit ? limit : ptx::kWaitLimitNs;
    p.drop_load = rt->drop_next_load.exchange(0) != 0;
    CUtensorMap ma, mw, mw2, mwh, mw2h, my;
    int rc = make_map_codes(&ma, P.a, P.a_stride, P.m, P.k, kHalf);
    if (rc == T0_OK) rc = make_map_codes(&mw, P.w[0], P.w_stride, P.n, P.k, kHalf);
    mw2 = mwh = mw2h = mw;
    if (rc == T0_OK && kGated) rc = make_map_codes(&mw2, P.w[1], P.w_stride, P.n, P.k, kHalf);
    if (p.whole < total) {
        if (rc == T0_OK) rc = make_map_codes(&mwh, P.w[0], P.w_stride, P.n, P.k, kHalf / 2);
        if (rc == T0_OK && kGated) rc = make_map_codes(&mw2h, P.w[1], P.w_stride, P.n, P.k, kHalf / 2);
    }
    if (rc != T0_OK) return rc;
    my = ma;
    // a TMA store writes whole 16 bytes: rows have to begin and end on such boundaries
    const uint64_t size = P.out_bf16 ? 2 : 4;
    if (((uintptr_t)P.y & 15) == 0 && P.y_stride * size % 16 == 0 && P.n * size % 16 == 0) {
        if ((rc = make_map_y(&my, P)) != T0_OK) return rc;
        p.tma_store = 1;
    }
    const cudaError_t e = gemm::launch_pdl(kern, 2 * (uint32_t)std::min<uint64_t>(items, (uint64_t)pairs), kThreads, smem_bytes(), rt->stream, ma, mw, mw2, mwh, mw2h, my, p);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "launch of the eight-bit product failed: %s", cudaGetErrorString(e));
    rt->launches.fetch_add(1);
    return T0_OK;
}

}  // namespace

int launch_pair(t0_runtime* rt, const Product& P, bool gated) {
    const DeviceGuard guard(rt->device);
    return gated ? launch_instance<true>(rt, P) : launch_instance<false>(rt, P);
}

}  // namespace q8
}  // namespace t0
