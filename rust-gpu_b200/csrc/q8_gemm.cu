// Products of rows in eight bits with weights in eight bits: the entries, and which kernel takes what.
#include <cmath>

#include "gemm_common.cuh"
#include "q8.cuh"
#include "runtime_internal.h"

namespace t0 {
namespace q8 {
namespace {

// Which kernel takes a product, and how it is cut: by a model of both kernels' times, its constants found over 430 shapes (1 .. 2200 rows, n 256 .. 16384, k 256 .. 14336, plain and gated; 20
// cuts each).  On those shapes the choice, with its bound on tiles, takes 3.6 % more time than each one's best on average and 44 % at most (gated 1015 x 500 x 13312: 27.8 us on pairs, 19.3 streamed; then 931 x 290 x 7711
// 19.0 / 13.6: gated tiles hold half the tokens, and the bound sends them to pairs from 769 rows on).  Shapes that the constants were not found on have not been measured; with weights beyond what L2 holds the
// rate that pairs are given is too high, and few rows go there (gated 48 x 8192 x 8192 30.0 on pairs, 24.3 streamed).  Nanoseconds, and bytes per nanosecond.  Both sides, plain, us on pairs / streamed:
// 128 x 4096 x 4096 12.4 / 9.3, 256 x 4096 x 4096 12.8 / 13.2, 512 x 4096 x 4096 13.0 / 16.2, 400 x 1024 x 4096 11.8 / 9.7, 1024 x 11008 x 4096 35.5 / 50.1.
//   streamed, a round of tiles: k blocks times the slowest of { issuing a block's copies and products, the weights' way from memory (slower with few CTAs), all operands' way from L2, the
//     products, one SM's way from L2 }, then the epilogue by its tokens, and the adding of parts;
//   pairs, a round: k blocks times the slower of { the products, the weights' way from memory }, and the epilogue; the last round may be one of half tiles.
float stream_time(const Product& P, uint32_t g, uint32_t tiles_m, const Cut& c, uint32_t clusters) {
    const uint32_t tiles = ceil_div(P.n, c.rows) * tiles_m, rounds = ceil_div(tiles, clusters), blocks = ceil_div(ceil_div(P.k, 128), c.parts);
    const float ctas = (float)std::min(tiles, clusters) * c.parts, w = g * c.rows * 128.0f, a = c.tokens * 128.0f;
    float block = g * (160.0f + 0.5f * c.tokens);
    block = std::max(block, ctas * w / tiles_m / 8000.0f / std::sqrt(std::sqrt(std::min(1.0f, ctas / 140.0f))));
    block = std::max(block, std::max(ctas * (w + a) / 21600.0f, (w + a) / 256.0f));
    block = std::max(block, 1.42f * g * c.tokens);
    const float parts = c.parts > 1 ? 1190.0f + 11.3f * g * c.tokens + 165.0f * (c.parts - 2) : 0.0f;
    return 2340.0f + rounds * (blocks * block + 7.29f * g * c.tokens + parts + (c.rows % 32 ? 187.0f : 0.0f));
}
float pair_time(const Product& P, uint32_t g, uint32_t pairs) {
    const uint64_t tiles_n = ceil_div(P.n, 256 / g), tiles = ceil_div(P.m, 256) * tiles_n, rest = tiles % pairs, halved = 2 * rest <= pairs ? rest : 0;
    const float blocks = (float)ceil_div(P.k, 128), rounds = (float)((tiles - halved + pairs - 1) / pairs);
    const float apart = P.a_stride % 128 || P.w_stride % 128 ? 1.23f : 1.0f;           // a row's 128 bytes lie in two lines
    const float whole = std::max(134.0f * apart, std::min<uint64_t>(std::min<uint64_t>(tiles, pairs), tiles_n) * 32768 / 12400.0f);
    const float half = std::max(171.0f * apart, std::min(halved, tiles_n) * 32768 / 12400.0f);
    return 6930.0f + rounds * (blocks * whole + 3220.0f) + (halved ? blocks * half : 0.0f);
}

Cut choose(const Product& P, bool gated, uint32_t sms) {
    const uint32_t g = gated ? 2 : 1, tiles_m = ceil_div(P.m, kMostTokens / g);
    Cut best = {0, 0, 0};
    if (tiles_m > 6) return best;                                          // streamed, the weights would be read that often (1985 x 896 x 1740 12.0 us, on pairs 9.5; 1145 x 2304 x 4096 15.4 and 17.1)
    const uint32_t* at_once = gemm_clusters_at_once();
    float least = pair_time(P, g, std::max(1u, sms / 2));
    for (uint32_t parts = 1; parts <= 4 && parts <= ceil_div(P.k, 128); ++parts) {
        const uint32_t clusters = std::max(1u, parts == 1 ? sms : at_once[parts]);
        const uint32_t even = ceil_div(P.n, std::max(1u, clusters / tiles_m));   // rows that make one round of everything
        for (const uint32_t rows : {even, 32u, 64u, 96u, 128u}) {
            if (rows > 128) continue;
            const Cut c = {std::max(8u, rows), (ceil_div(P.m, tiles_m) + 15) & ~15u, parts};
            const float t = stream_time(P, g, tiles_m, c, clusters);
            if (t < least) least = t, best = c;
        }
    }
    return best;
}

int launch(t0_runtime* rt, const Product& P, bool gated) {
    const DeviceGuard guard(rt->device);
    const Cut cut = choose(P, gated, (uint32_t)rt->sm_count);
    return cut.parts ? launch_stream(rt, P, gated, cut) : launch_pair(rt, P, gated);
}

// What both entries check; fills `P` but for the second matrix, the bias and the activation.
int check_product(uint64_t a, uint64_t a_scales, uint32_t* a_stride, uint64_t y, uint32_t* y_stride, uint32_t m, uint32_t n, uint32_t k, bool out_bf16, Product* P) {
    memset(P, 0, sizeof *P);
    const uint32_t size = out_bf16 ? 2 : 4;
    if (k == 0) return fail(T0_ERR_INVALID, "k must be positive");
    if (k > kMaxSum) return fail(T0_ERR_UNSUPPORTED, "k=%u: sums of more than %u products may leave 32 bits", k, kMaxSum);
    if (m > 0x40000000u || n > 0x40000000u) return fail(T0_ERR_INVALID, "m=%u, n=%u: at most 2^30", m, n);
    if (m == 0 || n == 0) return T0_OK;
    int rc = check_codes("a", a, a_scales, a_stride, k);
    if (rc != T0_OK) return rc;
    if (!y) return fail(T0_ERR_INVALID, "null device pointer");
    if (y % size) return fail(T0_ERR_INVALID, "y must be aligned to its numbers");
    if (*y_stride == 0) *y_stride = n;
    if (*y_stride < n) return fail(T0_ERR_INVALID, "y: a stride of %u numbers, rows have %u", *y_stride, n);
    P->a = (const int8_t*)a; P->a_scales = (const float*)a_scales; P->y = (void*)y;
    P->a_stride = *a_stride; P->y_stride = *y_stride;
    P->m = m; P->n = n; P->k = k; P->out_bf16 = out_bf16;
    if (touch(y, (uint64_t)n * size, (uint64_t)*y_stride * size, m, a, k, *a_stride, m) || touch(y, (uint64_t)n * size, (uint64_t)*y_stride * size, m, a_scales, 4, 4, m))
        return fail(T0_ERR_INVALID, "y overlaps a or its scales");
    return T0_OK;
}

int check_weights(const char* name, uint64_t w, uint64_t scales, uint32_t* stride, int which, Product* P) {
    const uint32_t size = P->out_bf16 ? 2 : 4;
    int rc = check_codes(name, w, scales, stride, P->k);
    if (rc != T0_OK) return rc;
    if (touch((uint64_t)P->y, (uint64_t)P->n * size, P->y_stride * size, P->m, w, P->k, *stride, P->n) ||
        touch((uint64_t)P->y, (uint64_t)P->n * size, P->y_stride * size, P->m, scales, (uint64_t)P->n * 4, (uint64_t)P->n * 4, 1))
        return fail(T0_ERR_INVALID, "y overlaps %s or its scales", name);
    P->w[which] = (const int8_t*)w; P->w_scales[which] = (const float*)scales;
    P->w_stride = *stride;
    return T0_OK;
}

}  // namespace
}  // namespace q8
}  // namespace t0

using namespace t0;
using namespace t0::q8;

extern "C" {

int t0_q8_gemm(t0_runtime* rt, const t0_q8_gemm_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_gemm_args a = *args;
    Product P;
    int rc = check_product(a.a, a.a_scales, &a.a_stride, a.y, &a.y_stride, a.m, a.n, a.k, a.out_bf16 != 0, &P);
    if (rc != T0_OK) return rc;
    if (a.m == 0 || a.n == 0) return check_rt(rt);
    if ((rc = check_weights("w", a.w, a.w_scales, &a.w_stride, 0, &P)) != T0_OK) return rc;
    if (a.bias & 3) return fail(T0_ERR_INVALID, "the bias must be 4-byte aligned");
    const uint64_t size = a.out_bf16 ? 2 : 4;
    if (touch(a.y, a.n * size, a.y_stride * size, a.m, a.bias, 4ull * a.n, 4ull * a.n, 1)) return fail(T0_ERR_INVALID, "y overlaps the bias");
    P.bias = (const float*)a.bias;
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    return launch(rt, P, false);
}

int t0_q8_gated(t0_runtime* rt, const t0_q8_gated_args* args) {
    if (!args) return fail(T0_ERR_INVALID, "null arguments");
    t0_q8_gated_args a = *args;
    Product P;
    int rc = check_product(a.a, a.a_scales, &a.a_stride, a.y, &a.y_stride, a.m, a.n, a.k, a.out_bf16 != 0, &P);
    if (rc != T0_OK) return rc;
    if (a.activation != T0_TEPI_RELU && a.activation != T0_TEPI_SILU && a.activation != T0_TEPI_GELU)
        return fail(T0_ERR_INVALID, "activation=%u: relu, silu or gelu", a.activation);
    if (a.m == 0 || a.n == 0) return check_rt(rt);
    if ((rc = check_weights("gate", a.gate, a.gate_scales, &a.w_stride, 0, &P)) != T0_OK) return rc;
    if ((rc = check_weights("up", a.up, a.up_scales, &a.w_stride, 1, &P)) != T0_OK) return rc;
    P.act = a.activation;
    if ((rc = check_rt(rt)) != T0_OK) return rc;
    return launch(rt, P, true);
}

}  // extern "C"
