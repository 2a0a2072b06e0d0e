// Attention of few rows (rows x group <= 16) over the paged four-bit cache: reading the cache once is all that counts.
//
// Transposed products on mma.sync: S^T = K Q^T with sixteen tokens as the rows of a tile and eight (row, head) columns, and O^T = V^T P^T
// with sixteen numbers of the head as rows.  Columns that no query fills cost a product nothing it would not cost anyway, and the cache's codes are
// the A operands of both: a nibble in the mantissa of a bf16 128 is 128 + code, so the codes of two neighbours become a register of the operand with a shift and a
// logical operation.  Steps and lows stay outside of the products:
//   score_j = a_j (q . (128 + c_j)) + b_j sum(q),   a_j = step_j, b_j = low_j - 128 step_j    (f32)
//   o       = sum_j (p_j step_j) (c_j - 8) + sum_j p_j (low_j + 8 step_j),   no p_j above 1
// where p_j step_j is rounded to bf16 (one rounding for each token and row, which a sum feels by at most 2^-8 of eight steps of the token's weight; the second sum stays f32).
// (The codes are centred before the product: 128 + c there, and 136 p_j step_j off the second sum, is 2.5 % faster, but the product's own sums then grow so far beyond their
// difference that an average of 4096 random values was off by 7e-3 in place of 2e-3.)
// A code is never an infinity or a NaN, so a token that a row must not see can be cut off by its factors alone, whatever its parameters are.
//
// The work is the list of all (sequence, key/value head) items' chunks of 64 tokens, cut into equal contiguous runs, one for each warp: whatever the lengths, every warp
// reads as much as the next.  A warp has its own two buffers, filled by bulk copies (the blocks of a chunk are contiguous pieces of the pages), and its own running
// maximum and sums.  Items that end up in several warps are joined, first inside the CTA, then between CTAs by the one that arrives last, always in order.
//
// 128 sequences of 5100 tokens on average, 8 key/value heads of 128 and 8 rows each (713 MB), take 156 to 167 us, 4.3 to 4.6 TB/s (109 us at the rate of a plain copy): 130 in chunks
// (5.5 TB/s), which the warps leave 10 us apart, 5 before, 5 of joins.  With three warps a scheduler of 168 registers the ALU is busy for 62 % of the cycles and an instruction issued
// in 57 %, most of them taking codes apart.  One row on 131072 tokens (143 MB) takes 44 us: 7 until a warp has its first chunk, 26 of chunks, 4 of joins, and the launch.  32 sequences' five rows in a window of 1000, 16 heads of 64 (36 MB): 23.7 us, 4 before, 8 of
// chunks (3 or 4 a warp), 4 of joins, and the launch.  8, 10 or 11 warps and chunks of 32 tokens were slower; codes by way of fp16 (half the shifts) 3 % faster for keys, but values'
// weights leave its range.
#include "kv4_attention.cuh"

namespace t0 {
namespace kv4 {
namespace {

constexpr int kTok = 64;                                  // tokens of a chunk
constexpr int kStages = 2;
constexpr float kLag = 8.0f;                              // powers of two by which a score may exceed its row's maximum so far; weights are 2^(score - maximum - kLag),
                                                          // so that none is above one: a weight times a step near the end of f32's range is no infinity
constexpr uint32_t kManyParts = 4;                        // CTAs' parts that one warp joins; more are shared by a CTA's warps
constexpr uint32_t kMaxParts = kMaxCtas;                  // parts of one item: at most one for each CTA

template <int D> constexpr int stage_bytes() { return kTok * (D + 8); }
template <int D, int NT> constexpr int warps() { return D == 128 ? (NT == 1 ? 12 : 8) : (NT == 1 ? 16 : 12); }
template <int D, int NT> constexpr int record_floats() { return 8 * NT * (D + 2); }

// position of tile row r among the sixteen tokens of a tile: neighbouring rows, and every second row, then lie in both halves of the 32 banks
__device__ __forceinline__ int token_of(int r) { return r ^ ((r >> 1) & 1); }

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 128 + code of nibbles i and i + 4.  (x & mask) | k128 is one instruction where one of the two constants is in a register: k128, made by keep().
__device__ __forceinline__ uint32_t keep(uint32_t x) {
    asm volatile("" : "+r"(x));
    return x;
}
__device__ __forceinline__ uint32_t codes_128(uint32_t w, int i, uint32_t k128) {
    uint32_t x;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(x) : "r"(w >> (4 * i)), "r"(k128));
    return x;
}
// code - 8, exactly
__device__ __forceinline__ uint32_t codes_centred(uint32_t w, int i, uint32_t k128) {
    const uint32_t x = codes_128(w, i, k128);
    const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&x, __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
    return *(const uint32_t*)&r;
}
// two f32 at once
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&p;
}

// The chunks of every sequence, in order, and how they are cut: made by the CTA for itself.
struct Plan {
    uint32_t prefix[1024 + 1];       // chunks (one head's) before the sequences that each thread looked at
    uint32_t warp_sum[32];
    uint32_t per_thread;             // sequences that one thread looked at
};

// chunks of sequence b for one head; rows it is to be left out for have none
__device__ __forceinline__ uint32_t chunks_of(const Attention& P, const Sequence& s) {
    if (s.rows == 0 || (uint32_t)s.rows * P.group > P.few) return 0;
    const int lo = first_seen(s, P.window) / kTok, hi = (s.len + kTok - 1) / kTok;
    return hi > lo ? hi - lo : 1;                         // at least one: rows that see nothing are written too
}

struct Item {
    uint32_t b, head;
    Sequence s;
    uint32_t chunks, c0;             // chunks of the item; the first chunk's number in the sequence
    uint32_t first;                  // its first unit
};

template <int kThreads>
__device__ __forceinline__ uint32_t make_plan(const Attention& P, Plan& plan) {
    const uint32_t n = P.B.n_seqs, per = (n + kThreads - 1) / kThreads, tid = threadIdx.x;
    uint32_t mine = 0;
    for (uint32_t b = tid * per; b < min(n, (tid + 1) * per); ++b) mine += chunks_of(P, sequence(P.B, b));
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if ((tid & 31) >= d) upto += other;
    }
    if ((tid & 31) == 31) plan.warp_sum[tid / 32] = upto;
    __syncthreads();
    const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, (tid & 31) < tid / 32 ? plan.warp_sum[tid & 31] : 0);
    plan.prefix[tid + 1] = before + upto;
    if (tid == 0) {
        plan.prefix[0] = 0;
        plan.per_thread = per;
    }
    __syncthreads();
    return plan.prefix[kThreads] * P.B.n_kv_heads;           // (less than 2^31: checked on the host)
}

// The item that unit u belongs to (u < all units).  By a whole warp, for one u: two votes in place of nine dependent steps took 0.5 us off the smallest call (8.0 us) and
// 1.4 off one whose warps have three or four chunks each (25.0).
template <int kThreads>
__device__ __forceinline__ Item item_of(const Attention& P, const Plan& plan, uint32_t u) {
    const uint32_t H = P.B.n_kv_heads;
    constexpr uint32_t kStep = kThreads / 32;             // the last thread whose prefix does not exceed u: the step of 32, then the place in it
    static_assert(kStep <= 32 && kThreads % 32 == 0);
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = (__popc(__ballot_sync(0xFFFFFFFFu, plan.prefix[lane * kStep] * H <= u)) - 1) * kStep;
    lo += __popc(__ballot_sync(0xFFFFFFFFu, lane < kStep && plan.prefix[lo + min(lane, kStep - 1)] * H <= u)) - 1;
    Item it;
    it.b = lo * plan.per_thread;
    uint32_t at = plan.prefix[lo] * H;
    for (;; ++it.b) {
        it.s = sequence(P.B, it.b);
        it.chunks = chunks_of(P, it.s);
        const uint32_t next = at + it.chunks * H;
        if (u < next || it.b + 1 >= P.B.n_seqs) break;
        at = next;
    }
    it.chunks = max(it.chunks, 1u);
    it.head = (u - at) / it.chunks;
    it.first = at + it.head * it.chunks;
    it.c0 = first_seen(it.s, P.window) / kTok;
    return it;
}

// The parts of one item, in order: records of the CTA's warps (record `from`, then the first ones of the warps behind), or of CTAs (the second one of the first, then the first ones).
struct Parts {
    const float* const* here;        // null: records of CTAs
    int from;
    const float* of_ctas;            // ... the second record of the first CTA
    uint32_t floats;                 // ... of a record
    uint32_t n;
    __device__ __forceinline__ const float* operator[](uint32_t i) const {
        if (here) return here[i == 0 ? from : 2 * (from / 2 + (int)i)];
        return of_ctas + (i == 0 ? 0 : (int64_t)(2 * i - 1) * floats);
    }
};

// Maximum and sum of the parts of an item, by one warp, for this lane's column (lane % kCols), and each part's weight: a row of `weight` for each.
template <int D, int NT>
__device__ __forceinline__ void weigh_parts(const Parts& parts, float (*weight)[8 * NT], float* top, float* sum) {
    constexpr int kCols = 8 * NT;
    constexpr uint32_t kEach = 32 / kCols;
    const uint32_t lane = threadIdx.x % 32, col = lane % kCols;
    float m = -INFINITY, l = 0.0f;
    for (uint32_t i = lane / kCols; i < parts.n; i += kEach) m = fmaxf(m, parts[i][kCols * D + col]);
#pragma unroll
    for (uint32_t d = kCols; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    const float base = m == -INFINITY ? 0.0f : m;
    for (uint32_t i = lane / kCols; i < parts.n; i += kEach) {
        const float* r = parts[i] + kCols * D + col;
        const float w = exp2_fast(r[0] - base);
        l += w * r[kCols];
        weight[i][col] = w;
    }
#pragma unroll
    for (uint32_t d = kCols; d < 32; d *= 2) l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
    __syncwarp();
    *top = m;
    *sum = l;
}

// The parts of an item added up by one warp: four numbers of every 128 for a lane.
template <int D, int NT>
__device__ __forceinline__ void add_parts(const Parts& parts, float (*weight)[8 * NT], float* top, float* sum, float4 (&total)[8 * NT * D / 128]) {
    constexpr int kPieces = 8 * NT * D / 128;
    const uint32_t lane = threadIdx.x % 32;
    weigh_parts<D, NT>(parts, weight, top, sum);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) total[j] = make_float4(0, 0, 0, 0);
#pragma unroll 2
    for (uint32_t i = 0; i < parts.n; ++i) {
        const float4* r = (const float4*)parts[i] + lane;
        float4 x[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) x[j] = r[32 * j];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const float f = weight[i][(128 * j + 4 * lane) / D];
            total[j].x = fmaf(f, x[j].x, total[j].x); total[j].y = fmaf(f, x[j].y, total[j].y);
            total[j].z = fmaf(f, x[j].z, total[j].z); total[j].w = fmaf(f, x[j].w, total[j].w);
        }
    }
    __syncwarp();
}

// numbers e .. e + 3 of an item's result; columns that are no row's are passed over
template <int D>
__device__ __forceinline__ void store(const Attention& P, const Item& it, uint32_t e, float4 x, float f) {
    const uint32_t c = e / D;
    if (c >= (uint32_t)it.s.rows * P.group) return;
    __nv_bfloat16* y = P.y + (uint64_t)(it.s.first_row + c / P.group) * P.y_stride + (it.head * P.group + c % P.group) * D + e % D;
    *(uint2*)y = make_uint2(pack(x.x * f, x.y * f), pack(x.z * f, x.w * f));
}
// What this lane's column (lane % kCols) is multiplied with.  A row with a token sees that token at least, so a sum of zero there has scores of minus infinity alone and makes the row NaN;
// a row without one is zeros.
template <int kCols>
__device__ __forceinline__ float inverse_of(const Attention& P, const Item& it, float sum) {
    return threadIdx.x % kCols < max(it.s.rows - it.s.len, 0) * P.group ? 0.0f : 1.0f / sum;
}
template <int D, int NT>
__device__ __forceinline__ void finish(const Attention& P, const Item& it, const float4 (&total)[8 * NT * D / 128], float sum) {
    const uint32_t lane = threadIdx.x % 32;
    const float inverse = inverse_of<8 * NT>(P, it, sum);
#pragma unroll
    for (int j = 0; j < 8 * NT * D / 128; ++j) {
        const uint32_t e = 128 * j + 4 * lane;
        store<D>(P, it, e, total[j], __shfl_sync(0xFFFFFFFFu, inverse, e / D));
    }
}

template <int D, int NT>
struct Params {
    Attention P;
    float* records;                  // one for each warp of the grid, then two for each CTA
    int* counters;                   // one for each CTA: parts that have arrived of the item it begins and does not end
    uint32_t min_warps;
};

template <int D, int NT>
__global__ void __launch_bounds__(warps<D, NT>() * 32, 1) kv4_decode_kernel(const __grid_constant__ Params<D, NT> G) {
    constexpr int kWarps = warps<D, NT>(), kThreads = kWarps * 32, kCols = 8 * NT;
    constexpr int kKeyWords = D / 32, kSteps = D / 16;    // words of a row in a lane; k steps of the scores
    constexpr int kValueWords = D / 64;
    constexpr int kRecord = record_floats<D, NT>();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Plan plan;
    __shared__ __align__(8) uint64_t bars[kWarps * kStages];
    __shared__ int abort_flag, rec_there[2 * kWarps], rec_open[2 * kWarps];
    __shared__ uint32_t many_parts[2], many_from[2];
    __shared__ Item many_item[2];
    __shared__ Item first_item, last_item[kWarps];         // the item that the CTA begins in, and those that the warps' runs end in
    __shared__ float weight_here[3 * kWarps][kCols], weight_of[2][kMaxParts][kCols];       // joining: of the parts in the CTA, and of CTAs' parts
    __shared__ const float* rec_at[2 * kWarps];
    const Attention& P = G.P;
    const Batch& B = P.B;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint32_t ring = ptx::smem_u32(smem) + warp * kStages * stage_bytes<D>();
    const uint8_t* ring_ptr = smem + warp * kStages * stage_bytes<D>();
    const uint32_t bar = ptx::smem_u32(bars) + warp * kStages * 8;
    if (threadIdx.x == 0) abort_flag = many_parts[0] = many_parts[1] = 0;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) ptx::mbar_init(bar + 8 * i, 1);
        ptx::fence_barrier_init();
    }
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const uint32_t units = make_plan<kThreads>(P, plan);
    if (units == 0) return;
    // how many warps of a CTA work: all, or fewer where that spreads the chunks over more SMs
    const uint32_t per_cta = min((uint32_t)kWarps, max(G.min_warps, (units + gridDim.x - 1) / gridDim.x));
    const uint32_t workers = min(units, gridDim.x * per_cta), whole = units / workers, rest = units % workers;
    const uint32_t me = blockIdx.x * per_cta + warp;
    const bool active = warp < per_cta && me < workers;
    auto start_of = [&](uint32_t w) { return w * whole + w * rest / workers; };       // w units / workers, rounded down
    auto worker_of = [&](uint32_t u) { return (uint32_t)(((uint64_t)(u + 1) * workers + units - 1) / units - 1); };
    if (blockIdx.x * per_cta >= workers) return;
    const uint32_t here = min(per_cta, workers - blockIdx.x * per_cta);               // warps of this CTA that work
    if (lane == 0) {
        rec_there[2 * warp] = rec_there[2 * warp + 1] = 0;
        rec_open[2 * warp] = rec_open[2 * warp + 1] = 0;
    }

    bool ok = true;
    if (active) {
        const uint32_t begin = start_of(me), end = start_of(me + 1);
        const uint32_t pl = B.page_log2, page_mask = (1u << pl) - 1;
        // ---- copies: chunk u of the run into stage s; item and chunk of the copies run ahead of the ones worked on.  A stage is laid out as a block of
        // 64 tokens whatever the page size, so that its addresses are constants: a block of fewer tokens is copied in four pieces, one for each lane.
        const Item ahead_first = item_of<kThreads>(P, plan, begin);
        Item ahead = ahead_first;
        uint32_t ahead_c = begin - ahead.first, ahead_left = end - begin;
        const uint32_t piece = lane & 3, piece_row = piece < 2 ? D / 2 : 4;                     // bytes of a token in this lane's piece
        const uint32_t piece_src = (piece == 0 ? 0 : piece == 1 ? D / 2 : piece == 2 ? D : D + 4) << pl, piece_dst = (piece == 0 ? 0 : piece == 1 ? D / 2 : piece == 2 ? D : D + 4) * kTok;
        auto issue = [&](int s) {                          // the next chunk of the run, if there is one
            if (ahead_left == 0) return;
            if (ahead_c == ahead.chunks) {
                ahead = item_of<kThreads>(P, plan, ahead.first + ahead.chunks);
                ahead_c = 0;
            }
            const uint32_t first = (ahead.c0 + ahead_c) * kTok;
            const uint32_t left = ahead.s.len > (int)first ? min((uint32_t)ahead.s.len - first, (uint32_t)kTok) : 0;
            const uint32_t blocks = (left + page_mask) >> pl;
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar + 8 * s, blocks * ((D + 8) << pl));
            __syncwarp();
            const uint32_t mine = pl == 6 ? lane : lane >> 2;
            if (mine < blocks) {
                const uint8_t* src = block_to_read<D>(B, ahead.b, (first >> pl) + mine, ahead.head);
                if (pl == 6) ptx::bulk_load(ring + s * stage_bytes<D>(), src, stage_bytes<D>(), bar + 8 * s);
                else ptx::bulk_load(ring + s * stage_bytes<D>() + piece_dst + ((mine * piece_row) << pl), src + piece_src, piece_row << pl, bar + 8 * s);
            }
            ++ahead_c;
            --ahead_left;
        };
        for (int s = 0; s < kStages; ++s) issue(s);

        uint32_t qf[NT][kSteps][2];                        // the queries' fragments
        float2 q_sum[NT];                                  // sums of the columns that this lane's scores are of
        float o[NT][D / 16][4], m[NT][2];
        float2 l[NT], low[NT];
        Item it = ahead_first;
        int p_row[NT][2];                                  // the tokens of those columns' rows

        auto begin_item = [&]() {
            const uint32_t cols = (uint32_t)it.s.rows * P.group;
            float part[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t col = 8 * n + g;
                const bool real = col < cols;
                const uint32_t row = real ? col / P.group : 0, head = it.head * P.group + (real ? col % P.group : 0);
                const uint4* src = (const uint4*)(P.q + (uint64_t)(it.s.first_row + row) * P.q_stride + head * D + t * (D / 4));
                part[n] = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint4 w = real ? src[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        qf[n][2 * i + j / 2][j % 2] = x[j];
                        part[n] += __uint_as_float(x[j] << 16) + __uint_as_float(x[j] & 0xFFFF0000u);
                    }
                }
                part[n] += __shfl_xor_sync(0xFFFFFFFFu, part[n], 1);
                part[n] += __shfl_xor_sync(0xFFFFFFFFu, part[n], 2);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    (i ? q_sum[n].y : q_sum[n].x) = __shfl_sync(0xFFFFFFFFu, part[n], 4 * (2 * t + i));
                    const uint32_t c = 8 * n + 2 * t + i;
                    p_row[n][i] = it.s.len - it.s.rows + (int)min(c / P.group, (uint32_t)it.s.rows - 1);
                    m[n][i] = -INFINITY;
                }
                l[n] = low[n] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[n][i][j] = 0.0f;
            }
        };

        const uint32_t k128 = keep(0x43004300u);
        const uint32_t key_at = token_of(g) * (D / 2) + t * (D / 8), param_at = D * kTok + 4 * token_of(g);
        const uint32_t value_at = kTok * (D / 2) + token_of(2 * t) * (D / 2) + g * (D / 16);
        // `whole`: every row sees every token of the chunk
        auto work_on = [&](const uint8_t* stage, int first, auto whole) {
            constexpr bool kWhole = decltype(whole)::value;
            float2 x[NT][kTok / 16][2];
            uint32_t v_param[kTok / 16][2];
#pragma unroll
            for (int i = 0; i < kTok / 16; ++i) {
                uint32_t wa[kKeyWords], wb[kKeyWords];
                const uint8_t* row = stage + key_at + i * (16 * D / 2);
                if constexpr (D == 128) {
                    const uint4 a = *(const uint4*)row, b = *(const uint4*)(row + 8 * (D / 2));
                    wa[0] = a.x; wa[1] = a.y; wa[2] = a.z; wa[3] = a.w;
                    wb[0] = b.x; wb[1] = b.y; wb[2] = b.z; wb[3] = b.w;
                } else {
                    const uint2 a = *(const uint2*)row, b = *(const uint2*)(row + 8 * (D / 2));
                    wa[0] = a.x; wa[1] = a.y;
                    wb[0] = b.x; wb[1] = b.y;
                }
                float acc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const uint32_t a0 = codes_128(wa[s / 2], 2 * (s % 2), k128), a1 = codes_128(wb[s / 2], 2 * (s % 2), k128);
                    const uint32_t a2 = codes_128(wa[s / 2], 2 * (s % 2) + 1, k128), a3 = codes_128(wb[s / 2], 2 * (s % 2) + 1, k128);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_bf16(acc[n], a0, a1, a2, a3, qf[n][s][0], qf[n][s][1]);
                }
                // scores, in powers of two
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t p = *(const uint32_t*)(stage + param_at + 4 * (16 * i + 8 * r));
                    v_param[i][r] = *(const uint32_t*)(stage + param_at + 4 * (kTok + 16 * i + 8 * r));
                    const float a = param_step(p) * P.scale_log2, b = fmaf(-128.0f, a, param_low(p) * P.scale_log2);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        x[n][i][r] = fma2(make_float2(acc[n][2 * r], acc[n][2 * r + 1]), make_float2(a, a), mul2(make_float2(b, b), q_sum[n]));
                    if constexpr (!kWhole) {
                        const int j = first + 16 * i + 8 * r + token_of(g);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (j > p_row[n][0] || (P.window && j <= p_row[n][0] - (int)P.window)) x[n][i][r].x = -INFINITY;
                            if (j > p_row[n][1] || (P.window && j <= p_row[n][1] - (int)P.window)) x[n][i][r].y = -INFINITY;
                        }
                    }
                }
            }
            // the maximum moves where a lane finds it left behind
            float2 top[NT];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                top[n] = make_float2(-INFINITY, -INFINITY);
#pragma unroll
                for (int i = 0; i < kTok / 16; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        top[n].x = fmaxf(top[n].x, x[n][i][r].x);
                        top[n].y = fmaxf(top[n].y, x[n][i][r].y);
                    }
                moved |= top[n].x > m[n][0] + kLag || top[n].y > m[n][1] + kLag;
            }
            if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) {
                        top[n].x = fmaxf(top[n].x, __shfl_xor_sync(0xFFFFFFFFu, top[n].x, d));
                        top[n].y = fmaxf(top[n].y, __shfl_xor_sync(0xFFFFFFFFu, top[n].y, d));
                    }
                    top[n] = make_float2(fmaxf(top[n].x, m[n][0]), fmaxf(top[n].y, m[n][1]));
                    const float2 less = make_float2(m[n][0] == top[n].x ? 1.0f : exp2_fast(m[n][0] - top[n].x), m[n][1] == top[n].y ? 1.0f : exp2_fast(m[n][1] - top[n].y));
                    m[n][0] = top[n].x;
                    m[n][1] = top[n].y;
                    l[n] = mul2(l[n], less);
                    low[n] = mul2(low[n], less);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        o[n][i][0] *= less.x; o[n][i][1] *= less.y;
                        o[n][i][2] *= less.x; o[n][i][3] *= less.y;
                    }
                }
            }
            // weights, and the values' steps in them
            uint32_t pf[NT][kTok / 16][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 minus = make_float2(m[n][0] == -INFINITY ? 0.0f : -m[n][0] - kLag, m[n][1] == -INFINITY ? 0.0f : -m[n][1] - kLag);
#pragma unroll
                for (int i = 0; i < kTok / 16; ++i)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float step = param_step(v_param[i][r]), base = fmaf(8.0f, step, param_low(v_param[i][r]));
                        const float2 y = add2(x[n][i][r], minus), p = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                        l[n] = add2(l[n], p);
                        float2 w = mul2(p, make_float2(step, step));
                        if constexpr (kWhole) {
                            low[n] = fma2(p, make_float2(base, base), low[n]);
                        } else {                           // the parameters of what is not seen may be anything
                            if (x[n][i][r].x == -INFINITY) w.x = 0.0f; else low[n].x = fmaf(p.x, base, low[n].x);
                            if (x[n][i][r].y == -INFINITY) w.y = 0.0f; else low[n].y = fmaf(p.y, base, low[n].y);
                        }
                        pf[n][i][r] = transpose8x8(pack(w.x, w.y));
                    }
            }
            // values
#pragma unroll
            for (int i = 0; i < kTok / 16; ++i) {
                uint32_t w[4][kValueWords];
#pragma unroll
                for (int r = 0; r < 4; ++r) {              // (token_of(2 t + 1) is token_of(2 t) + 1 or - 1)
                    const int away = (r & 1) ? (t & 1 ? -(D / 2) : D / 2) : 0;
                    const uint8_t* row = stage + value_at + away + (16 * i + 8 * (r >> 1)) * (D / 2);
                    if constexpr (D == 128) {
                        const uint2 a = *(const uint2*)row;
                        w[r][0] = a.x; w[r][1] = a.y;
                    } else {
                        w[r][0] = *(const uint32_t*)row;
                    }
                }
#pragma unroll
                for (int j = 0; j < kValueWords; ++j) {
                    const uint32_t even0 = __byte_perm(w[0][j], w[1][j], 0x5410), odd0 = __byte_perm(w[0][j], w[1][j], 0x7632);
                    const uint32_t even1 = __byte_perm(w[2][j], w[3][j], 0x5410), odd1 = __byte_perm(w[2][j], w[3][j], 0x7632);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t a0 = codes_centred(even0, k, k128), a1 = codes_centred(odd0, k, k128), a2 = codes_centred(even1, k, k128), a3 = codes_centred(odd1, k, k128);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_bf16(o[n][4 * j + k], a0, a1, a2, a3, pf[n][i][0], pf[n][i][1]);
                    }
                }
            }
        };

        // the item is done as far as this warp goes: sums over the lanes, then to y, or to a record
        auto end_item = [&](bool opens, bool goes_on, bool last) {
            float sum[NT][2], rest[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    sum[n][k] = k ? l[n].y : l[n].x;
                    rest[n][k] = k ? low[n].y : low[n].x;
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) {
                        sum[n][k] += __shfl_xor_sync(0xFFFFFFFFu, sum[n][k], d);
                        rest[n][k] += __shfl_xor_sync(0xFFFFFFFFu, rest[n][k], d);
                    }
                }
            if (opens && !goes_on) {
                const uint32_t cols = (uint32_t)it.s.rows * P.group;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t c = 8 * n + 2 * t + k;
                        if (c >= cols) continue;
                        __nv_bfloat16* to = P.y + (uint64_t)(it.s.first_row + c / P.group) * P.y_stride + (it.head * P.group + c % P.group) * D + g * (D / 8);
                        const float inverse = p_row[n][k] < 0 ? 0.0f : 1.0f / sum[n][k];         // (as inverse_of)
                        uint32_t out[D / 16];
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) out[i] = pack((o[n][i][k] + rest[n][k]) * inverse, (o[n][i][2 + k] + rest[n][k]) * inverse);
#pragma unroll
                        for (int i = 0; i < D / 64; ++i) *(uint4*)(to + 8 * i) = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
                    }
                return;
            }
            const uint32_t which = opens ? 1 : 0;          // 0: begun before this run, 1: begun in it
            // after the last chunk of the run the warp's buffers are free; before, the record has to go out
            float* rec = last ? (float*)ring_ptr : G.records + (uint64_t)(blockIdx.x * kWarps + warp) * kRecord;
            if (last) __syncwarp();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t c = 8 * n + 2 * t + k;
                    float4* to = (float4*)(rec + c * D + g * (D / 8));
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
                        to[i] = make_float4(o[n][2 * i][k] + rest[n][k], o[n][2 * i][2 + k] + rest[n][k], o[n][2 * i + 1][k] + rest[n][k], o[n][2 * i + 1][2 + k] + rest[n][k]);
                    if (g == 0) {
                        rec[kCols * D + c] = m[n][k];
                        rec[kCols * D + kCols + c] = sum[n][k];
                    }
                }
            if (lane == 0) {
                rec_there[2 * warp + which] = 1;
                rec_open[2 * warp + which] = goes_on;
                rec_at[2 * warp + which] = rec;
            }
        };

        if (warp == 0 && lane == 0) first_item = it;
        uint32_t u = begin, phase = 0;
        while (u < end) {
            if (u != begin) it = item_of<kThreads>(P, plan, u);
            const uint32_t item_end = it.first + it.chunks;
            const bool opens = u == it.first;
            begin_item();
            for (; u < end && u < item_end; ++u) {
                const int s = (u - begin) % kStages;
                ok = ok && ptx::mbar_wait_warp(bar + 8 * s, (phase >> s) & 1, &abort_flag, P.wait_limit_ns);
                if (!ok) break;
                phase ^= 1u << s;
                const int first = (int)(it.c0 + (u - it.first)) * kTok, p_first = it.s.len - it.s.rows;
                const uint8_t* stage = ring_ptr + s * stage_bytes<D>();
                if (first + kTok - 1 <= p_first && (P.window == 0 || first > it.s.len - 1 - (int)P.window)) work_on(stage, first, std::true_type{});
                else work_on(stage, first, std::false_type{});
                __syncwarp();
                issue(s);
            }
            if (!ok) break;
            end_item(opens, u < item_end, u == end);
        }
        if (lane == 0) last_item[warp] = it;
        if (!ok) {                                         // copies in flight end before the CTA does
            for (int s = 0; s < kStages; ++s) {
                volatile int never = 0;
                ptx::mbar_wait_warp(bar + 8 * s, (phase >> s) & 1, &never, P.wait_limit_ns);
            }
            if (lane == 0) *(volatile int*)P.timeout_status = kStatusProducerTimeout | (int)blockIdx.x;
        }
    }
    __syncthreads();
    if (abort_flag) return;

    // ---- joining.  A record a warp begins in (index 2 w) continues what the warp before has as the record it ends in (2 w + 1), or, where the warp lies in the item as a
    // whole, as its own 2 w.  So a run of parts of one item is the record 2 a + 1 (or 0), then 2 (a + 1), 2 (a + 2), ... to the one that is not open.  Every run is one warp's,
    // all at the same time.  At most two are open, at the CTA's begin and at its end: they become records of the CTA, and the CTA that arrives last finishes the item.
    float* const cta_records = G.records + (uint64_t)gridDim.x * kWarps * kRecord;
    auto join = [&](int from, const Item& it) {              // the run that begins with record `from`
        Parts parts = {rec_at, from, nullptr, 0, 1};
        bool open = rec_open[from] != 0;
        for (uint32_t w = from / 2 + 1; open && w < here; ++w, ++parts.n) open = rec_open[2 * w] != 0;
        float top, sum;
        float4 total[kCols * D / 128];
        add_parts<D, NT>(parts, weight_here + from, &top, &sum, total);
        const uint32_t k = from & 1;                          // 0: begun before the CTA's run, 1: in it
        if (k == 0 || open) {
            float* to = cta_records + (uint64_t)(2 * blockIdx.x + k) * kRecord;
#pragma unroll
            for (int j = 0; j < kCols * D / 128; ++j) ((float4*)to)[32 * j + lane] = total[j];
            if (lane < kCols) {
                to[kCols * D + lane] = top;
                to[kCols * D + kCols + lane] = sum;
            }
            const uint32_t first_cta = worker_of(it.first) / per_cta, n = worker_of(it.first + it.chunks - 1) / per_cta - first_cta + 1;
            __threadfence();
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0) before = (uint32_t)atomicAdd(G.counters + first_cta, 1);
            if (__shfl_sync(0xFFFFFFFFu, before, 0) != n - 1) return;
            if (lane == 0) G.counters[first_cta] = 0;
            __threadfence();
            if (n > kManyParts) {                           // a long item: the CTA's warps share it, below
                if (lane == 0) {
                    many_parts[k] = n;
                    many_from[k] = first_cta;
                    many_item[k] = it;
                }
                return;
            }
            parts = Parts{nullptr, 0, cta_records + (uint64_t)(2 * first_cta + 1) * kRecord, kRecord, n};
            add_parts<D, NT>(parts, weight_of[k], &top, &sum, total);
        }
        finish<D, NT>(P, it, total, sum);
    };
    if (warp < here && rec_there[2 * warp + 1]) join(2 * warp + 1, last_item[warp]);
    if (rec_there[0]) {
        // the run of record 0 goes to a warp that has none, the first warp if they all do
        const uint32_t idle = __ballot_sync(0xFFFFFFFFu, lane < kWarps && (lane >= here || !rec_there[2 * min(lane, (uint32_t)kWarps - 1) + 1]));
        if (warp == (idle ? (uint32_t)__ffs(idle) - 1 : 0u)) join(0, first_item);
    }
    __syncthreads();
    for (int k = 0; k < 2; ++k) {
        const uint32_t n = many_parts[k];
        if (n == 0) continue;
        // every warp weighs all parts for itself, and adds up the 128 numbers of a record that are its own
        const Parts parts = {nullptr, 0, cta_records + (uint64_t)(2 * many_from[k] + 1) * kRecord, kRecord, n};
        float top, sum;
        weigh_parts<D, NT>(parts, weight_of[k], &top, &sum);
        __syncthreads();                                    // (the same weights from every warp)
        const Item it = many_item[k];
        const float inverse = inverse_of<kCols>(P, it, sum);
        for (uint32_t e = 128 * warp + 4 * lane; e < kCols * D; e += 128 * kWarps) {
            float4 total = make_float4(0, 0, 0, 0);
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) {
                const float4 x = *(const float4*)(parts[i] + e);
                const float f = weight_of[k][i][e / D];
                total.x = fmaf(f, x.x, total.x); total.y = fmaf(f, x.y, total.y); total.z = fmaf(f, x.z, total.z); total.w = fmaf(f, x.w, total.w);
            }
            store<D>(P, it, e, total, __shfl_sync(0xFFFFFFFFu, inverse, e / D));
        }
    }
}

template <int D, int NT>
int launch(const Attention& p, uint32_t sms, cudaStream_t stream) {
    constexpr int smem = warps<D, NT>() * kStages * stage_bytes<D>();
    static bool attr_set[64] = {};   // per instantiation, per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return fail(T0_ERR_CUDA, "cudaFuncSetAttribute(smem=%d): %s", smem, cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    Params<D, NT> g;
    g.P = p;
    g.counters = (int*)p.scratch;
    g.records = (float*)(p.scratch + kv4_counter_bytes());
    g.min_warps = 4;
    const cudaError_t e = gemm::launch_pdl(kv4_decode_kernel<D, NT>, std::min(sms, kMaxCtas), warps<D, NT>() * 32, smem, stream, g);
    if (e != cudaSuccess) return fail(T0_ERR_CUDA, "attention launch failed: %s", cudaGetErrorString(e));
    return T0_OK;
}

}  // namespace

// a multiple of 128
size_t decode_scratch_bytes(uint32_t sms) {
    const size_t n = std::min(sms, kMaxCtas);
    auto one = [&](size_t warps, size_t record) { return ((n * warps + 2 * n) * record * sizeof(float) + 127) / 128 * 128; };
    return std::max(std::max(one(warps<128, 1>(), record_floats<128, 1>()), one(warps<128, 2>(), record_floats<128, 2>())),
                    std::max(one(warps<64, 1>(), record_floats<64, 1>()), one(warps<64, 2>(), record_floats<64, 2>())));
}

int launch_decode(const Attention& p, uint32_t head_dim, uint32_t columns, uint32_t sms, cudaStream_t stream) {
    if (head_dim == 128) return columns <= 8 ? launch<128, 1>(p, sms, stream) : launch<128, 2>(p, sms, stream);
    return columns <= 8 ? launch<64, 1>(p, sms, stream) : launch<64, 2>(p, sms, stream);
}

}  // namespace kv4
}  // namespace t0
