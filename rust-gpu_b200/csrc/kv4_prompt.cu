// Attention of many rows (rows x group > 16) over the paged four-bit cache: tcgen05 products, the cache's codes made bf16 on the way into shared memory.
//
// An item is 256 rows (pairs of token and query head of one key/value head, two tiles of 128) against the chunks of 128 tokens that any of them sees.  Per chunk
//   S = Q K^T (shared memory x shared memory -> tensor memory),  P = 2^(S - m) (one thread a row),  O += P V (P in tensor memory, over S's own columns)
// half a chunk at a time: the 512 columns of tensor memory are O of both tiles and, for each, S of two halves, so that the scores of one half are there when the softmax
// warps are done with the other.  The maximum only moves when it is left behind by more than 2^8 (then O is read, scaled and written back), so that O is rarely touched; weights are taken
// against 2^8 times the maximum, so that none is above one and a sum of them and of values leaves f32 only where a sum against the true maximum could.
//   warps 0-3, 4-7  softmax of tile 0 and 1, and their results     warps 8-11   codes -> bf16, K and V into rings of two stages
//   warp 12         issues the products                            warps 13-15  queries of the next item into shared memory
// Keys, values and weights are rounded to bf16 for the products (step * code + low, once; the sums of weights are of unrounded ones): a score feels that by at most 2^-8 of
// sum |q k|, a result by 2^-8 of sum p |v| for each of weights and values.  Results of random numbers are off by 4.4e-3 of their size, 1.7e-3 of which is their own rounding.
// Keys and queries in fp16, kept in range by powers of two for each chunk and row, brought that to 2.8e-3 and took 4 to 18 % longer: the powers have to be agreed on by
// all warps that make a chunk's keys before the first is stored.  A value row that is NaN is put in as zeros and
// its key as NaN: a row that sees the token becomes NaN through its score, a row that must not see it has weight 0, and 0 x 0 adds nothing.  For the same reason a value
// whose rounding to bf16 would be an infinity is bf16's largest number here.
//
// The units of work are all items' chunks, and kItemUnits for what an item costs beside them, in equal contiguous runs, one for each CTA.  Items whose chunks end up in
// several CTAs leave parts (O, m, l) that a second kernel joins.
//
// 8192 tokens on themselves, 32 query and 8 key/value heads of 128, take 595 us, 925 TFLOP/s of what the mask leaves (heads of 64: 438 us, before the clock falls); 2048 behind 8192 others 328 us.  A chunk takes a CTA 3700
// clocks, of which the products need 2048 and the powers of two 2048 (a scheduler makes four a clock): the softmax warps work for 2800 of them and wait for the rest.  Over
// more than a few launches the clock falls from 1965 to 1725 MHz at the board's 1000 W (534 us before that), so that less work in one unit saves little: no scores in one
// product a chunk (610 us), maxima of three numbers (600), a quarter of the powers by a polynomial (605) nor eight warps for the codes were faster; without the codes'
// work altogether 544.
#include "kv4_attention.cuh"

namespace t0 {
namespace kv4 {
namespace {

constexpr int kTok = 128, kRows = 256, kTile = 128;
constexpr int kDequantWarps = 4;
constexpr int kThreads = (12 + kDequantWarps) * 32;
constexpr uint32_t kIssuer = 8 + kDequantWarps;           // the warp that issues the products
constexpr uint32_t kItemUnits = 3;                        // an item's queries, results and idle times in chunks' time (10600 of 3800 clocks, measured on a prompt of 8192 tokens with heads
                                                          // of 128; with heads of 64, a mixed batch of 24 sequences took 217 us, 222 with 1 here)
constexpr float kLag = 8.0f;                              // powers of two by which a score may exceed its row's maximum so far; weights are 2^(score - maximum - kLag)

template <int D> constexpr uint32_t tile_bytes() { return kTile * D * 2; }
template <int D> constexpr uint32_t smem_bytes() { return 6 * tile_bytes<D>() + 1024 + 512; }
template <int D> constexpr uint32_t record_floats() { return kRows * (D + 2); }          // [D][256] sums, [256] maxima, [256] sums of weights

// The items of one head in the order (sequence, tile), and their chunks: what every thread found in its share, summed up.
struct Plan {
    uint32_t tiles[kThreads + 1];    // tiles before the sequences of each thread
    uint32_t units[kThreads + 1];    // units before the tiles of each thread
    uint32_t warp_sum[kThreads / 32];
    uint32_t seqs_each, tiles_each;
};

__device__ __forceinline__ uint32_t tiles_of(const Attention& P, const Sequence& s) {
    const uint32_t n = (uint32_t)s.rows * P.group;
    return n <= P.few ? 0 : (n + kRows - 1) / kRows;
}

struct Item {
    Sequence s;
    uint32_t b, tile, head;
    int c0, c1;                      // its chunks
    __device__ __forceinline__ uint32_t units() const { return (uint32_t)(c1 - c0) + kItemUnits; }
    __device__ __forceinline__ void range(const Attention& P) {
        const int i0 = (int)(tile * kRows / P.group), i1 = min(s.rows - 1, (int)((tile * kRows + kRows - 1) / P.group));
        const int p0 = s.len - s.rows + i0, p1 = s.len - s.rows + i1;
        c0 = P.window && p0 >= (int)P.window ? (p0 - (int)P.window + 1) / kTok : 0;
        c1 = p1 < 0 ? c0 + 1 : p1 / kTok + 1;             // at least one, also where no row sees anything: its rows are written
    }
    // the next tile; sequences that have none here are passed over
    __device__ __forceinline__ void advance(const Attention& P) {
        if (++tile >= tiles_of(P, s)) {
            tile = 0;
            for (uint32_t i = 0; i < P.B.n_seqs; ++i) {
                if (++b == P.B.n_seqs) {
                    b = 0;
                    ++head;
                }
                s = sequence(P.B, b);
                if (tiles_of(P, s)) break;
            }
        }
        range(P);
    }
};

__device__ __forceinline__ uint32_t scan(uint32_t mine, uint32_t* warp_sum, uint32_t* out) {
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if ((threadIdx.x & 31) >= d) upto += other;
    }
    if ((threadIdx.x & 31) == 31) warp_sum[threadIdx.x / 32] = upto;
    __syncthreads();
    const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, (threadIdx.x & 31) < threadIdx.x / 32 ? warp_sum[threadIdx.x & 31] : 0);
    out[threadIdx.x + 1] = before + upto;
    if (threadIdx.x == 0) out[0] = 0;
    __syncthreads();
    return out[kThreads];
}
__device__ __forceinline__ uint32_t last_not_above(const uint32_t* prefix, uint32_t x) {
    uint32_t lo = 0, hi = kThreads;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (prefix[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}
// tile number `at` of one head
__device__ __forceinline__ Item tile_at(const Attention& P, const Plan& plan, uint32_t at) {
    const uint32_t th = last_not_above(plan.tiles, at);
    Item it;
    it.head = 0;
    it.b = th * plan.seqs_each;
    uint32_t n = plan.tiles[th];
    for (;; ++it.b) {
        it.s = sequence(P.B, it.b);
        const uint32_t next = n + tiles_of(P, it.s);
        if (at < next || it.b + 1 >= P.B.n_seqs) break;
        n = next;
    }
    it.tile = at - n;
    it.range(P);
    return it;
}
// returns the units of one head
__device__ __forceinline__ uint32_t make_plan(const Attention& P, uint32_t most, Plan& plan) {
    const uint32_t n = P.B.n_seqs, each = (n + kThreads - 1) / kThreads, tid = threadIdx.x;
    if (tid == 0) plan.seqs_each = each;
    uint32_t mine = 0;
    for (uint32_t b = tid * each; b < min(n, (tid + 1) * each); ++b) mine = min(mine + tiles_of(P, sequence(P.B, b)), most + 1);
    const uint32_t tiles = scan(mine, plan.warp_sum, plan.tiles);
    if (tiles > most) return 0;
    const uint32_t tiles_each = (tiles + kThreads - 1) / kThreads;
    if (tid == 0) plan.tiles_each = tiles_each;
    mine = 0;
    if (tid * tiles_each < tiles) {
        Item it = tile_at(P, plan, tid * tiles_each);
        for (uint32_t i = tid * tiles_each;;) {
            mine += it.units();
            if (++i >= min(tiles, (tid + 1) * tiles_each)) break;
            it.advance(P);
        }
    }
    return scan(mine, plan.warp_sum, plan.units);
}
// the item that unit u (of all heads) belongs to, and the unit it begins with
__device__ __forceinline__ Item item_of(const Attention& P, const Plan& plan, uint32_t per_head, uint32_t u, uint32_t* first) {
    const uint32_t head = u / per_head, at = u % per_head, th = last_not_above(plan.units, at);
    Item it = tile_at(P, plan, th * plan.tiles_each);
    uint32_t n = plan.units[th];
    while (at >= n + it.units()) {
        n += it.units();
        it.advance(P);
    }
    it.head = head;
    *first = head * per_head + n;
    return it;
}
// where run c of `runs` begins: units * c / runs, rounded down.  There are no more runs than units, so that none is empty.
__device__ __forceinline__ uint32_t start_of(uint32_t c, uint32_t units, uint32_t runs) { return c * (units / runs) + c * (units % runs) / runs; }

// A run's way through its items: the chunks c .. c + n - 1 of one after the other.
struct Walk {
    Item it;
    uint32_t first, end;             // the item's first unit; the run's end
    int c;
    uint32_t n;                      // 0: the run is over
    __device__ __forceinline__ void count() {
        const int upto = (int)min(end - first, it.units()) - (int)kItemUnits;
        n = max(it.c0 + upto - c, 0);
    }
    __device__ __forceinline__ Walk(const Attention& P, const Plan& plan, uint32_t per_head, uint32_t begin, uint32_t end_) : end(end_) {
        it = item_of(P, plan, per_head, begin, &first);
        c = it.c0 + max((int)(begin - first) - (int)kItemUnits, 0);
        count();
    }
    __device__ __forceinline__ void next(const Attention& P) {
        first += it.units();
        n = 0;
        if (first >= end) return;
        it.advance(P);
        c = it.c0;
        count();
    }
};

// What the joining kernel needs to know of the item that a CTA's run begins in.
struct Cut {
    uint32_t units, first, chunks;   // of the launch; the item's first, and its chunks (0: the run is empty)
    uint32_t tile, head;
    int first_row;
    uint32_t total;                  // rows x group of the sequence
    int first_token;                 // of its first row
};

struct Params {
    Attention P;
    float* records;                  // two for each CTA: of the item it begins in, of the item it ends in
    Cut* cuts;                       // one for each CTA
    // Sequences whose rows do not overlap have no more tiles than this (2^23 at most), and their units fit into 32 bits.  Where row_start is not ascending, which
    // sequence() reports, there may be more: then none is taken.
    uint32_t most_tiles;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&p;
}
// infinities (of finite parameters, so positive ones) made bf16's largest number; a NaN stays one
__device__ __forceinline__ uint32_t bounded(uint32_t x) {
    const __nv_bfloat162 v = __hmin2_nan(*(const __nv_bfloat162*)&x, __nv_bfloat162(__ushort_as_bfloat16(0x7F7F), __ushort_as_bfloat16(0x7F7F)));
    return *(const uint32_t*)&v;
}
// Whether the largest value that a row's parameters allow, 15 step + low, leaves bf16 where the parameters are finite.
__device__ __forceinline__ bool leaves_bf16(uint32_t params) {
    const __nv_bfloat16 top = __hfma(__ushort_as_bfloat16(0x4170), __ushort_as_bfloat16((uint16_t)params), __ushort_as_bfloat16((uint16_t)(params >> 16)));
    return __bfloat16_as_ushort(top) == 0x7F80;
}
template <int D>
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const __grid_constant__ Params G) {
    constexpr uint32_t kTileBytes = tile_bytes<D>(), kPanel = kTile * 128, kTmem = 512;
    constexpr uint32_t kS = 0, kO = 2 * kTok;             // columns of tensor memory: S of both tiles (P over them), O of both
    extern __shared__ uint8_t smem_raw[];
    __shared__ Plan plan;
    const Attention& P = G.P;
    const Batch& B = P.B;
    const uint32_t warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + 6 * kTileBytes);
    const uint32_t q_smem = ptx::smem_u32(smem), k_smem = q_smem + 2 * kTileBytes, v_smem = k_smem + 2 * kTileBytes, bar = ptx::smem_u32(bars);
    // barriers
    const uint32_t q_full = bar, q_empty = bar + 8, drained = bar + 16;
    auto k_full = [&](uint32_t s) { return bar + 24 + 8 * s; };
    auto k_empty = [&](uint32_t s) { return bar + 40 + 8 * s; };
    auto v_full = [&](uint32_t s) { return bar + 56 + 8 * s; };
    auto v_empty = [&](uint32_t s) { return bar + 72 + 8 * s; };
    auto s_full = [&](uint32_t t, uint32_t half) { return bar + 88 + 16 * t + 8 * half; };
    auto p_full = [&](uint32_t t, uint32_t half) { return bar + 120 + 16 * t + 8 * half; };
    // The sums of one more half are in O: waited for only where O is scaled, by a warp that has not yet given the next half's weights away, so that no more than the phase it
    // asks for can be open or over.  The end of an item has a barrier of its own: two phases may end there before a warp looks.
    auto o_step = [&](uint32_t t) { return bar + 152 + 8 * t; };
    auto o_full = [&](uint32_t t) { return bar + 168 + 8 * t; };
    uint32_t* tmem_holder = (uint32_t*)(bars + 23);
    volatile int* abort_flag = (volatile int*)(tmem_holder + 1);
    if (threadIdx.x == 0) {
        ptx::mbar_init(q_full, 3);
        ptx::mbar_init(q_empty, 1);
        ptx::mbar_init(drained, 1);
        for (uint32_t s = 0; s < 2; ++s) {
            ptx::mbar_init(k_full(s), kDequantWarps);
            ptx::mbar_init(k_empty(s), 1);
            ptx::mbar_init(v_full(s), kDequantWarps);
            ptx::mbar_init(v_empty(s), 1);
            for (uint32_t half = 0; half < 2; ++half) {
                ptx::mbar_init(s_full(s, half), 1);
                ptx::mbar_init(p_full(s, half), 4);
            }
            ptx::mbar_init(o_step(s), 1);
            ptx::mbar_init(o_full(s), 1);
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
    }
    if (warp == kIssuer) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_holder), kTmem);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_holder, 0);
    ptx::grid_launch_dependents();
    // Behind kv4_decode in one call too, whose rows and scratch are others: without this wait nothing says that what an append before both wrote is visible here.  (Beginning beside that
    // kernel, and waiting at the end, took 218.2 us in place of 220.8 for a batch of 24 sequences of both kinds; with a word that it releases and this one acquires, 221.7.)
    ptx::grid_dependency_wait();

    const uint32_t per_head = make_plan(P, G.most_tiles, plan), units = per_head * B.n_kv_heads, runs = min(gridDim.x, units);
    const uint32_t begin = blockIdx.x < runs ? start_of(blockIdx.x, units, runs) : 0, end = blockIdx.x < runs ? start_of(blockIdx.x + 1, units, runs) : 0;
    bool ok = true;
    auto wait = [&](uint32_t b, uint32_t parity) {
        if (ok) ok = ptx::mbar_wait_warp(b, parity, abort_flag, P.wait_limit_ns);
        return ok;
    };
    if (begin >= end && threadIdx.x == 0) G.cuts[blockIdx.x] = Cut{};
    if (begin < end) {
        Walk walk(P, plan, per_head, begin, end);
        const Item& it = walk.it;
        if (threadIdx.x == 0)
            G.cuts[blockIdx.x] = Cut{units, walk.first, (uint32_t)(it.c1 - it.c0), it.tile, it.head, it.s.first_row, (uint32_t)it.s.rows * P.group, it.s.len - it.s.rows};

        if (warp < 8) {
            // ------------------------------------------------------------ softmax: a thread has a row
            const uint32_t t = warp / 4, r = threadIdx.x & 127, lanes = ((warp & 3) * 32) << 16;
            const uint32_t s_col = tmem + kS + t * kTok + lanes, o_col = tmem + kO + t * D + lanes;
            uint32_t s_phase = 0, o_phase = 0, halves = 0;             // halves this tile has had
            for (; ok && walk.n; walk.next(P)) {
                const int c = walk.c;
                const uint32_t n = walk.n, total = (uint32_t)it.s.rows * P.group;
                const bool opens = c == it.c0, closes = c + (int)n == it.c1;
                const uint32_t row = it.tile * kRows + t * kTile + r;
                if (it.tile * kRows + t * kTile < total) {
                    const int last = (int)min(row, total - 1);
                    const int p = it.s.len - it.s.rows + last / (int)P.group;                      // the row's token
                    const int p_low = it.s.len - it.s.rows + (int)((it.tile * kRows + t * kTile) / P.group);     // the tile's first and last
                    const int p_high = it.s.len - it.s.rows + (int)(min(it.tile * kRows + t * kTile + kTile, total) - 1) / (int)P.group;
                    float m = -INFINITY;
                    float2 l[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                    for (uint32_t i = 0; i < 2 * n; ++i) {
                        const uint32_t half = i & 1, col = s_col + 64 * half;
                        if (!wait(s_full(t, half), s_phase)) break;
                        s_phase ^= half;
                        ptx::tc_fence_after_sync();
                        const int first = c * kTok + (int)i * 64;
                        const bool whole = first + 63 <= p_low && (P.window == 0 || first > p_high - (int)P.window);
                        float x[64];
                        ptx::tmem_ld_32x32b_x32(col, *(uint32_t(*)[32])x);
                        ptx::tmem_ld_32x32b_x32(col + 32, *(uint32_t(*)[32])(x + 32));
                        ptx::tmem_ld_wait();
                        if (!whole) {
                            const int from = P.window ? p - (int)P.window + 1 - first : -1, to = p - first;      // columns the row sees
#pragma unroll
                            for (int j = 0; j < 64; ++j)
                                if (j < from || j > to) x[j] = -INFINITY;
                        }
                        float tops[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) tops[j] = x[16 * j];
#pragma unroll
                        for (int j = 1; j < 16; ++j)
#pragma unroll
                            for (int k = 0; k < 4; ++k) tops[k] = fmaxf(tops[k], x[16 * k + j]);
                        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * P.scale_log2;         // (the scale is positive)
                        const bool left_behind = top > m + kLag || (m == -INFINITY && top > m);
                        if (__any_sync(0xFFFFFFFFu, left_behind)) {          // once or twice an item
                            const float m_new = left_behind ? ceilf(top) : m, less = m == m_new ? 1.0f : exp2_fast(m - m_new);
                            m = m_new;
                            l[0] = __fmul2_rn(l[0], make_float2(less, less));
                            l[1] = __fmul2_rn(l[1], make_float2(less, less));
                            // O has to be at rest: the sums of the half before the last are done (these scores were issued behind them), those of the last are waited for
                            if (i > 0) {
                                if (!wait(o_step(t), (halves - 1) & 1)) break;
                                ptx::tc_fence_after_sync();
                            }
#pragma unroll 1
                            for (int k = 0; i > 0 && k < D / 8; ++k) {
                                uint32_t o[8];
                                ptx::tmem_ld_32x32b_x8(o_col + 8 * k, o);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * less);
                                ptx::tmem_st_32x32b_x8(o_col + 8 * k, o);
                            }
                        }
                        const float minus = m == -INFINITY ? 0.0f : -m - kLag;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t y[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float2 e = __ffma2_rn(make_float2(x[32 * k + 2 * j], x[32 * k + 2 * j + 1]), make_float2(P.scale_log2, P.scale_log2), make_float2(minus, minus));
                                const float2 w = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                                l[j % 2] = __fadd2_rn(l[j % 2], w);
                                y[j] = pack(w.x, w.y);
                            }
                            ptx::tmem_st_32x32b_x16(col + 16 * k, y);            // over columns that have been read
                        }
                        ptx::tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        ptx::mbar_arrive_if(p_full(t, half), lane == 0);
                        ++halves;
                    }
                    const float sum = (l[0].x + l[0].y) + (l[1].x + l[1].y);
                    if (!wait(o_full(t), o_phase)) break;
                    o_phase ^= 1;
                    ptx::tc_fence_after_sync();
                    if (opens && closes) {
                        const float inverse = p < 0 ? 0.0f : 1.0f / sum;         // a row with a token sees that: scores of minus infinity alone make it NaN
                        __nv_bfloat16* y = P.y + (uint64_t)(it.s.first_row + last / (int)P.group) * P.y_stride + (it.head * P.group + last % P.group) * D;
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) {
                            uint32_t x[32];
                            ptx::tmem_ld_32x32b_x32(o_col + 32 * q, x);
                            ptx::tmem_ld_wait();
                            if (row < total) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    uint32_t w[4];
#pragma unroll
                                    for (int k = 0; k < 4; ++k) w[k] = pack(__uint_as_float(x[8 * j + 2 * k]) * inverse, __uint_as_float(x[8 * j + 2 * k + 1]) * inverse);
                                    *(uint4*)(y + 32 * q + 8 * j) = make_uint4(w[0], w[1], w[2], w[3]);
                                }
                            }
                        }
                    } else {
                        float* rec = G.records + (uint64_t)(2 * blockIdx.x + (opens ? 1 : 0)) * record_floats<D>() + t * kTile + r;
#pragma unroll
                        for (int q = 0; q < D / 32; ++q) {
                            uint32_t x[32];
                            ptx::tmem_ld_32x32b_x32(o_col + 32 * q, x);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) rec[(32 * q + j) * kRows] = __uint_as_float(x[j]);
                        }
                        rec[D * kRows] = m;
                        rec[(D + 1) * kRows] = sum;
                    }
                    ptx::tc_fence_before_sync();           // the next item's first product writes O after this warp's next p_full
                }
            }
        } else if (warp < kIssuer) {
            // ------------------------------------------------------------ codes to bf16
            const uint32_t tid = threadIdx.x - 256, part = tid & 3;       // a quarter of rows tid / 4 + kRowStep i
            constexpr int kWords = D / 32;                                  // words of a quarter
            constexpr int kRowStep = kDequantWarps * 8, kEach = kTok / kRowStep;
            uint32_t k128;
            asm volatile("mov.b32 %0, 0x43004300;" : "=r"(k128));
            const uint32_t pl = B.page_log2;
            // places of the rows, the same in every chunk: their parameters and codes in a block, their 16-byte units in a stage.  The order in which a quarter's units are
            // stored differs between lanes, so that eight lanes hit all banks.
            uint32_t param_off[kEach], code_off[kEach], unit_off[kWords];
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint32_t slot = (tid / 4 + kRowStep * i) & ((1u << pl) - 1);
                param_off[i] = params_at<D>(pl, 0) + 4 * slot;
                code_off[i] = slot * (D / 2) + part * (D / 8);
            }
            const bool swapped = D == 128 && part >= 2;
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const uint32_t unit = part * kWords + (swapped ? j ^ 2 : j);
                unit_off[j] = unit / 8 * kPanel + tid / 4 * 128 + ((unit % 8 ^ (tid / 4 & 7)) << 4);
            }
            // A chunk's codes are asked for half a chunk's work before they are used, and its pages' numbers a whole one before that.  A page outside the cache is read
            // as page 0 and reported at the end; where there is no token page 0 is read too, and the parameters are zeros.
            Walk ahead = walk;
            uint32_t left_out = 0xFFFFFFFFu, next_pages[kEach];
            bool next_there[kEach], there[kEach];
            uint32_t next_head = 0, next_seq = 0, raw[2][kEach][kWords], kp[kEach], vp[kEach];
            const uint8_t* block[kEach];
            bool more = ahead.n != 0;                       // whether pages have been looked up that are not loaded yet
            auto look_up = [&]() {                          // of the chunk that is ahead, if there is one; then on to the next
                more = ahead.n != 0;
                if (!more) return;
                next_head = ahead.it.head;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const uint32_t token = (uint32_t)ahead.c * kTok + tid / 4 + kRowStep * i;
                    next_there[i] = token < (uint32_t)ahead.it.s.len;
                    next_pages[i] = next_there[i] ? (uint32_t)B.page_table[(uint64_t)ahead.it.b * B.table_stride + (token >> pl)] : 0;
                }
                next_seq = ahead.it.b;
                ++ahead.c;
                if (--ahead.n == 0) ahead.next(P);
            };
            auto load = [&](int which) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    if (which == 0) {
                        if (next_pages[i] >= B.n_pages) {
                            left_out = next_seq;
                            next_pages[i] = 0;
                        }
                        block[i] = B.pages + ((uint64_t)next_pages[i] * B.n_kv_heads + next_head) * ((D + 8) << pl);
                        there[i] = next_there[i];
                        kp[i] = *(const uint32_t*)(block[i] + param_off[i]);
                        vp[i] = *(const uint32_t*)(block[i] + param_off[i] + (4u << pl));
                    }
                    const uint8_t* src = block[i] + code_off[i] + (which ? (D / 2) << pl : 0);
                    if constexpr (kWords == 4) {
                        const uint4 w = *(const uint4*)src;
                        raw[which][i][0] = w.x; raw[which][i][1] = w.y; raw[which][i][2] = w.z; raw[which][i][3] = w.w;
                    } else {
                        const uint2 w = *(const uint2*)src;
                        raw[which][i][0] = w.x; raw[which][i][1] = w.y;
                    }
                }
            };
            auto store = [&](int which, uint32_t base, const uint32_t (&params)[kEach], bool far) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const __nv_bfloat162 step = twice(params[i] & 0xFFFFu), low = twice(params[i] >> 16);
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        const uint32_t w = swapped ? raw[which][i][(j ^ 2) % kWords] : raw[which][i][j];
                        const uint32_t v0 = value_of(w, 0, k128, step, low), v1 = value_of(w, 1, k128, step, low), v2 = value_of(w, 2, k128, step, low), v3 = value_of(w, 3, k128, step, low);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + unit_off[j] + i * (kRowStep * 128)), "r"(v0), "r"(v1), "r"(v2), "r"(v3) : "memory");
                    }
                }
                if (far) {                                  // hardly ever: over this thread's units once more, in a loop (bounds in the lines above, in a second copy of them, took 3 % of a mixed batch)
#pragma unroll 1
                    for (uint32_t n = 0; n < kEach * kWords; ++n) {
                        const uint32_t unit = part * kWords + n % kWords, at = base + unit / 8 * kPanel + (tid / 4 + n / kWords * kRowStep) * 128 + ((unit % 8 ^ (tid / 4 & 7)) << 4);
                        uint32_t v0, v1, v2, v3;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3) : "r"(at) : "memory");
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(bounded(v0)), "r"(bounded(v1)), "r"(bounded(v2)), "r"(bounded(v3)) : "memory");
                    }
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
            };
            look_up();
            bool at_hand = more;                            // whether there is a chunk whose codes are loaded
            if (at_hand) {
                load(0);
                load(1);
                look_up();
            }
            uint32_t stage = 0, phase = 0;
            while (ok && at_hand) {
                // parameters of this chunk; those of a NaN value go into its key
                uint32_t kq[kEach], vq[kEach];
                bool far = false;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const bool bad = (vp[i] & 0x7F800000u) == 0x7F800000u || (vp[i] & 0x7F80u) == 0x7F80u;
                    kq[i] = !there[i] ? 0u : bad ? 0x7FC07FC0u : kp[i];
                    vq[i] = !there[i] || bad ? 0u : vp[i];
                    far |= leaves_bf16(kq[i]) || leaves_bf16(vq[i]);
                }
                far = __any_sync(0xFFFFFFFFu, far);
                if (!wait(k_empty(stage), phase ^ 1)) break;
                store(0, k_smem + stage * kTileBytes, kq, far);
                ptx::mbar_arrive_if(k_full(stage), lane == 0);
                at_hand = more;
                if (more) load(0);
                if (!wait(v_empty(stage), phase ^ 1)) break;
                store(1, v_smem + stage * kTileBytes, vq, far);
                ptx::mbar_arrive_if(v_full(stage), lane == 0);
                if (more) {
                    load(1);
                    look_up();
                }
                stage ^= 1;
                phase ^= stage == 0;
            }
            if (left_out != 0xFFFFFFFFu) report(B, kStatusBadPage, left_out);
        } else if (warp == kIssuer) {
            // ------------------------------------------------------------ the products
            constexpr uint32_t kIdescS = ptx::make_idesc_bf16_f32(kTile, 64, 0), kIdescO = ptx::make_idesc_bf16_f32(kTile, D, 1), kHalf = 64 * 128 / 16;
            const uint32_t issue = ptx::elect_one();
            uint32_t k_count = 0, v_count = 0, q_phase = 0, p_phase[2] = {0, 0};        // chunks of K and V so far; stages and phases follow from them
            auto scores = [&](uint32_t t, uint32_t half) {
                const uint32_t a = ptx::smem_desc_lo(q_smem + t * kTileBytes, 16), b = ptx::smem_desc_lo(k_smem + (k_count & 1) * kTileBytes, 16) + half * kHalf;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = (k / 4) * (kPanel / 16) + (k % 4) * 2;
                    ptx::umma_bf16_ss_if(issue, tmem + kS + t * kTok + half * 64, a + at, b + at, kIdescS, k > 0);
                }
                ptx::umma_commit_if(issue, s_full(t, half));
            };
            auto sums = [&](uint32_t t, uint32_t half, bool more) {
                const uint32_t b = ptx::smem_desc_lo(v_smem + (v_count & 1) * kTileBytes, kPanel) + half * kHalf;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    ptx::umma_bf16_ts_mn_if(issue, tmem + kO + t * D, tmem + kS + t * kTok + half * 64 + k * 8, b + k * 128, kIdescO, k > 0 || more);
                ptx::umma_commit_if(issue, o_step(t));
            };
            for (; ok && walk.n; walk.next(P)) {
                const uint32_t n = walk.n, total = (uint32_t)it.s.rows * P.group;
                const uint32_t tiles = it.tile * kRows + kTile < total ? 2 : 1;
                if (!wait(q_full, q_phase) || !wait(k_full(k_count & 1), (k_count >> 1) & 1)) break;
                q_phase ^= 1;
                ptx::tc_fence_after_sync();
                for (uint32_t half = 0; half < 2; ++half)
                    for (uint32_t t = 0; t < tiles; ++t) scores(t, half);
                ptx::umma_commit_if(issue, k_empty(k_count & 1));
                ++k_count;
                if (n == 1) ptx::umma_commit_if(issue, q_empty);
                for (uint32_t i = 0; i < 2 * n && ok; ++i) {   // sums of half i, then scores of half i + 2 in the same columns
                    const uint32_t half = i & 1, c = i / 2;
                    const bool more = c + 1 < n;
                    if (half == 0) {
                        if (!wait(v_full(v_count & 1), (v_count >> 1) & 1)) break;
                        if (more && !wait(k_full(k_count & 1), (k_count >> 1) & 1)) break;
                    }
                    for (uint32_t t = 0; t < tiles && ok; ++t) {
                        if (!wait(p_full(t, half), p_phase[t])) break;
                        p_phase[t] ^= half;
                        ptx::tc_fence_after_sync();
                        sums(t, half, i > 0);
                        if (i + 1 == 2 * n) ptx::umma_commit_if(issue, o_full(t));
                        if (more) scores(t, half);
                    }
                    if (!ok || half == 0) continue;
                    ptx::umma_commit_if(issue, v_empty(v_count & 1));
                    ++v_count;
                    if (more) {
                        ptx::umma_commit_if(issue, k_empty(k_count & 1));
                        ++k_count;
                        if (c + 2 == n) ptx::umma_commit_if(issue, q_empty);
                    }
                }
            }
            // what is in flight ends before the memory it uses is given back: in a run that went well the last sums have been waited for by the softmax warps
            if (!ok) {
                volatile int never = 0;
                ptx::umma_commit_if(issue, drained);
                ptx::mbar_wait_warp(drained, 0, &never, P.wait_limit_ns);
            }
        } else if (warp > kIssuer) {
            // ------------------------------------------------------------ queries: a lane has the same 16 bytes of every sixth (twelfth) row
            constexpr uint32_t kLanes = D / 8, kStep = 3 * 32 / kLanes;
            const uint32_t unit = lane % kLanes, r0 = (warp - kIssuer - 1) * (32 / kLanes) + lane / kLanes;
            const uint32_t step_i = kStep / P.group, step_g = kStep % P.group;
            uint32_t phase = 1;
            for (; ok && walk.n; walk.next(P)) {
                const uint32_t total = (uint32_t)it.s.rows * P.group, base = it.tile * kRows;
                if (!wait(q_empty, phase)) break;
                phase ^= 1;
                const uint32_t rows = total - base <= kTile ? kTile : kRows;
                uint32_t i = (base + r0) / P.group, g = (base + r0) % P.group;
                const __nv_bfloat16* q = P.q + (uint64_t)it.s.first_row * P.q_stride + it.head * P.group * D + unit * 8;
                for (uint32_t r = r0; r < rows; r += kStep) {
                    const bool there = base + r < total;
                    cp_async16(q_smem + (r / kTile) * kTileBytes + (unit / 8) * kPanel + (r % kTile) * 128 + (((unit % 8) ^ (r & 7)) << 4),
                               there ? q + i * P.q_stride + g * D : q, there ? 16 : 0);
                    i += step_i;
                    g += step_g;
                    if (g >= P.group) {
                        g -= P.group;
                        ++i;
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                ptx::fence_proxy_async_smem();
                __syncwarp();
                ptx::mbar_arrive_if(q_full, lane == 0);
            }
        }
        if (!ok && lane == 0) atomicCAS(P.timeout_status, 0, (warp == kIssuer ? kStatusMmaTimeout : warp < 8 ? kStatusEpilogueTimeout : kStatusProducerTimeout) | (int)blockIdx.x);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == kIssuer) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, kTmem);
    }
}

// Joins the parts of the items whose chunks several CTAs of the launch before worked on: sum_i 2^(m_i - m) O_i over sum_i 2^(m_i - m) l_i, in order.  Bound by latency and by
// the reads of the parts (133 KB each, 39 MB at most, from L2): 17 us for all 148 CTAs' by itself, from cold.  Block (c, z): the item that the boundary before CTA c cuts, if c is the first one
// to cut it; z: a slice of its rows.  A thread has a row and a quarter of its numbers.
constexpr int kJoinRows = 64, kJoinThreads = kJoinRows * 4;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv4_prompt_join_kernel(const __grid_constant__ Params G) {
    const Attention& P = G.P;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const uint32_t slices = kRows / kJoinRows, c = blockIdx.x / slices + 1, z = blockIdx.x % slices;
    const Cut cut = G.cuts[c];
    if (cut.chunks == 0) return;
    const uint32_t runs = min(gridDim.x / slices + 1, cut.units);
    const uint32_t at = start_of(c, cut.units, runs), chunk0 = cut.first + kItemUnits, behind = chunk0 + cut.chunks;
    if (at <= chunk0 || start_of(c - 1, cut.units, runs) > chunk0) return;      // all chunks lie in this run, or an earlier boundary cuts them
    if (cut.tile * kRows + z * kJoinRows >= cut.total) return;
    const uint32_t r = z * kJoinRows + threadIdx.x % kJoinRows, part = threadIdx.x / kJoinRows, row = cut.tile * kRows + r;
    constexpr int kEach = D / 4;
    auto record = [&](uint32_t i) { return G.records + (uint64_t)(2 * i + (i == c - 1 ? 1 : 0)) * record_floats<D>() + r; };
    float top = -INFINITY, l = 0.0f, sum[kEach] = {};
    uint32_t parts_end = c;                                // the run behind the last one with a part
    while (parts_end < runs && start_of(parts_end, cut.units, runs) < behind) ++parts_end;
    for (uint32_t i = c - 1; i < parts_end; ++i) top = fmaxf(top, record(i)[D * kRows]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 1
    for (uint32_t i = c - 1; i < parts_end; ++i) {
        const float* rec = record(i);
        const float w = exp2_fast(rec[D * kRows] - base);
        l = fmaf(w, rec[(D + 1) * kRows], l);
#pragma unroll
        for (int j = 0; j < kEach; ++j) sum[j] = fmaf(w, rec[(part * kEach + j) * kRows], sum[j]);
    }
    if (row >= cut.total) return;
    const float inverse = row < max(-cut.first_token, 0) * P.group ? 0.0f : 1.0f / l;
    __nv_bfloat16* y = P.y + (uint64_t)(cut.first_row + row / P.group) * P.y_stride + (cut.head * P.group + row % P.group) * D + part * kEach;
#pragma unroll
    for (int j = 0; j < kEach / 8; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = pack(sum[8 * j + 2 * k] * inverse, sum[8 * j + 2 * k + 1] * inverse);
        *(uint4*)(y + 8 * j) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int D>
int launch(const Attention& p, uint32_t sms, cudaStream_t stream) {
    constexpr int smem = smem_bytes<D>();
    static bool attr_set[64] = {};   // per instantiation, per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_prompt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return fail(T0_ERR_CUDA, "cudaFuncSetAttribute(smem=%d): %s", smem, cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    Params g;
    g.P = p;
    g.cuts = (Cut*)(p.scratch + kv4_counter_bytes() + decode_scratch_bytes(sms));
    g.most_tiles = (uint32_t)((uint64_t)p.B.n_rows * p.group / kRows) + p.B.n_seqs;
    g.records = (float*)(g.cuts + kMaxCtas);
    const uint32_t ctas = std::min(sms, kMaxCtas);
    cudaError_t e = gemm::launch_pdl(kv4_prompt_kernel<D>, ctas, kThreads, smem, stream, g);
    if (e == cudaSuccess && ctas > 1) e = gemm::launch_pdl(kv4_prompt_join_kernel<D>, (ctas - 1) * (kRows / kJoinRows), kJoinThreads, 0, stream, g);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "attention launch failed: %s", cudaGetErrorString(e));
    return T0_OK;
}

}  // namespace

size_t prompt_scratch_bytes(uint32_t sms) { return kMaxCtas * sizeof(Cut) + (size_t)2 * std::min(sms, kMaxCtas) * record_floats<128>() * sizeof(float); }

int launch_prompt(const Attention& p, uint32_t head_dim, uint32_t sms, cudaStream_t stream) {
    return head_dim == 128 ? launch<128>(p, sms, stream) : launch<64>(p, sms, stream);
}

}  // namespace kv4
}  // namespace t0
