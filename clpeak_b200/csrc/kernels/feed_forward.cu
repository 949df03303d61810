// The products of a gated feed-forward layer: both projections with the activation, their gradients, and products of 8-bit
// integers with scales for each token and channel.
//
//   forward    g = x Wg^T, u = x Wu^T, h = act(g) * u
//   backward   dg = dh * u * act'(g), du = dh * act(g);  dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//   8 bits     c = float(sum of int8 products) * a_scale * b_scale + bias, and the forward pass with such sums
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "../clpk_activation.cuh"
#include "../clpk_internal.h"
#include "../clpk_pair.cuh"
#include "../clpk_ptx.cuh"

namespace clpk {

#include "../clpk_linear.cuh"
#include "../clpk_linear_few.cuh"

// ---- the products -------------------------------------------------------------------------------------------

struct Matrix {
    const void *base;
    uint64_t ld;                        // elements
};

// One product of a layer: sums over `k` of an m x n result.
struct Product {
    uint32_t m, n, k;
    Matrix a, b[2];                     // kGated: b[0] = Wg, b[1] = Wu
    void *c[3];                         // kGated: h, g, u
    uint64_t ldc;
    int out, activation;
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
    uint32_t *status;
};

constexpr uint32_t kMostRows = 0x7FFFFF00u;         // coordinates of whole tiles are signed 32-bit numbers

static uint64_t elem_bytes(int dtype) { return dtype == CLPK_DT_F32 ? 4 : dtype == CLPK_DT_I8 ? 1 : 2; }

// K blocks of 128 bytes
static uint32_t linear_k_blocks(uint32_t k, int dtype) { return (uint32_t)(((uint64_t)k * elem_bytes(dtype) + kRowBytesK - 1) / kRowBytesK); }

static uint32_t ceil_div(uint32_t a, uint32_t b) { return (a - 1) / b + 1; }

struct LinearPlan {
    uint32_t tn, splits;
};

// Clusters of `splits` pairs that the chip holds at a time: of a whole B200's 148 SMs, 33 of four CTAs that take an SM each and 15 of
// eight, as cudaOccupancyMaxActiveClusters counts them for every tile width.
static uint32_t linear_resident(uint32_t splits)
{
    const uint32_t pairs = (uint32_t)num_sms() / 2;
    return splits == 1 ? pairs : splits == 2 ? pairs * 33 / 74 : pairs * 15 / 74;
}

// Microseconds of linear_kernel besides its launch: `blocks` K blocks and `tiles` tiles one after another, with an exchange of
// partial sums where K is split.  Fitted to what 60 shapes of 131 to 8192 tokens took with every width and split, and 73 backward
// passes with every width and number of parts.
static float linear_estimate(float blocks, float tiles, uint32_t tn, uint32_t splits)
{
    const float wide = (float)tn / 256.0f;
    return blocks * (0.12f + 0.15f * wide) + tiles * (0.8f + 1.3f * wide + (splits > 1 ? 3.5f + 2.0f * wide : 0.0f));
}

// Tile width and K ranges: the cheapest by the estimate.  Of the 60 shapes it was fitted to it takes the fastest choice for
// 53, and the geometric mean is 0.6 % slower; of 60 others 59 are within 1 % of the fastest, and one is 3 % slower.
static LinearPlan plan_linear(const Product &w, LinearForm form, uint32_t k_blocks)
{
    const uint32_t cols = form == kGated ? 2 * w.n : w.n;
    LinearPlan plan = {256, 1};
    float best = 1e30f;
    for (uint32_t splits = 1; splits <= 4 && splits <= k_blocks; splits *= 2)
        for (uint32_t tn = 64; tn <= 256; tn += 64) {
            const uint64_t tiles = (uint64_t)ceil_div(w.m, kLinearM) * ceil_div(cols, tn);
            if (linear_resident(splits) == 0)
                continue;
            const float waves = (float)((tiles - 1) / linear_resident(splits) + 1);
            const float t = linear_estimate(waves * (float)ceil_div(k_blocks, splits), waves, tn, splits);
            if (t < best) {
                best = t;
                plan = {tn, splits};
            }
        }
    return plan;
}

// what a launch of linear_kernel has in common
template <int DT, LinearForm FORM, typename Maps, typename Params>
static int launch_linear_tiles(const Maps &maps, Params &p, LinearPlan plan, uint32_t n_tiles, const char *what, cudaStream_t s)
{
    p.tn = plan.tn;
    p.splits = plan.splits;
    const uint32_t clusters = plan.splits > 1 ? n_tiles : std::min(n_tiles, linear_resident(1));
    p.kps = linear_kps(plan.tn);
    p.stages = linear_stages(plan.tn);
    p.tmem_cols = 32;
    while (p.tmem_cols < (n_tiles > clusters ? 2 : 1) * plan.tn)
        p.tmem_cols *= 2;
    return launch_clusters(linear_kernel<DT, FORM>, what, clusters * 2 * plan.splits, kLinearThreads, p.stages * p.kps * linear_block_bytes(plan.tn) + kLinearFixedBytes, 2 * plan.splits, s, maps, p);
}

static LinearResult linear_result(void *base, uint64_t ld, uint32_t m, uint32_t n, int type)
{
    return {base, ld, m, n, n - n % (uint32_t)(16 / elem_bytes(type)), type};
}

template <int DT, LinearForm FORM>
static int launch_linear(const Product &w, uint32_t k_blocks, cudaStream_t s)
{
    const uint64_t elem = elem_bytes(DT);
    const LinearPlan plan = plan_linear(w, FORM, k_blocks);
    const uint32_t tile_cols = FORM == kGated ? plan.tn / 2 : plan.tn;
    LinearMaps maps = {};
    int rc = make_matrix_map(&maps.a, w.a.base, w.m, w.k * elem, w.a.ld * elem, 128);
    for (int i = 0; i < (FORM == kGated ? 2 : 1) && rc == CLPK_OK; i++)
        rc = make_matrix_map(&maps.b[i], w.b[i].base, w.n, w.k * elem, w.b[i].ld * elem, plan.tn / 2);
    LinearParams p = {};
    for (int i = 0; i < 3 && rc == CLPK_OK; i++)
        if (w.c[i]) {
            p.c[i] = linear_result(w.c[i], w.ldc, w.m, w.n, w.out);
            rc = make_result_map(&maps.c[i], p.c[i]);
        }
    if (rc != CLPK_OK)
        return rc;
    const uint32_t tiles_m = ceil_div(w.m, kLinearM), tiles_n = ceil_div(w.n, tile_cols);
    p.order = tile_order(tiles_m, tiles_n);
    p.k_blocks = k_blocks;
    p.activation = w.activation;
    p.keep = w.c[1] ? 1 : 0;
    p.a_scale = w.a_scale;
    p.b_scale = w.b_scale;
    p.u_scale = w.u_scale;
    p.bias = w.bias;
    p.status = w.status;
    return launch_linear_tiles<DT, FORM>(maps, p, plan, tiles_m * tiles_n, "linear", s);
}

template <LinearForm FORM> constexpr uint32_t few_cols = FORM == kGated ? 64 : 128;      // features of a tile

// K ranges of linear_few_kernel: as many as the chip holds CTAs for at once, as long as each has some blocks of K; with long sums
// also where that loads the SMs more evenly.  Fitted to 70 shapes of 1 to 64 tokens (1 % slower than the fastest in the
// geometric mean); over 70 others of up to 128 tokens, with few_tokens, it is 2.4 % slower, 53 are within 2 %, and the worst takes
// 49 us in one range where four would take 39 (64 x 10039 x 15855).  What it decides: int8 1 x 4096 x 4096 in one range 9.2 us, in
// four 5.2; 8 x 30080 x 4096 (235 tiles) 26.7, in two 23.0.
static uint32_t few_splits(uint32_t tokens, uint32_t tiles, uint32_t k_blocks, uint32_t sms)
{
    uint32_t splits = 1;
    if (k_blocks >= 8 && tiles * 2 <= sms)
        splits = 2;
    if ((k_blocks >= 48 && tiles > sms && tiles * 5 <= sms * 6) || (k_blocks >= 16 && tiles * 2 > sms * 3 && tiles < sms * 2))
        splits = 2;
    if (k_blocks >= (tokens >= 64 ? 4u : 8u) && tiles * 4 <= sms * 9 / 7)
        splits = 4;
    if (k_blocks >= 32 && tokens <= 48 && tiles * 2 > sms && tiles * 10 <= sms * 7)
        splits = 4;
    if (k_blocks >= 14 && tiles * 8 <= (k_blocks >= 64 ? sms : sms * 6 / 7))
        splits = 8;
    return splits;
}

// Whether the tokens are few: up to 64 they are; then it depends on whether finishing them or filling the chip costs more (96
// tokens: 15 tiles of 48 blocks 7.3 us here, 10.1 on pairs; 128 tokens: 12 of 50 9.4 and 13.4, 126 of 25 20.8 and 17.8, 4 of 4
// 6.4 and 5.0).
static bool few_tokens(uint32_t tokens, uint32_t tiles, uint32_t k_blocks, uint32_t sms)
{
    if (tokens <= 64)
        return true;
    if (tokens <= 96)
        return k_blocks < 36 || tiles * 5 <= sms * 3;
    return tokens <= 128 && k_blocks >= 20 && few_splits(tokens, tiles, k_blocks, sms) >= 4;
}

// How linear_few_kernel is launched: K ranges, the ring, and where the partial sums lie.
static void plan_few(FewParams &p, uint32_t tiles, uint32_t sms)
{
    p.tokens = (p.m + 15) / 16 * 16;
    p.tmem_cols = 32;
    while (p.tmem_cols < p.tokens)
        p.tmem_cols *= 2;
    p.splits = few_splits(p.m, tiles, p.k_blocks, sms);
    // as many CTAs as an SM gets share its memory; a ring has two stages at least, and is as large as the sums
    const uint32_t stage_bytes = kHalfTileBytes + p.tokens * kRowBytesK, sums = p.splits * ((p.m + p.splits - 1) / p.splits) * kFewRows * 4;
    uint32_t each = std::min((tiles * p.splits - 1) / sms + 1, (uint32_t)kFewResident), budget = 0;
    if ((each == 2 || (each == 1 && p.k_blocks < 32 * p.splits)) && 227 * 1024 / (each + 1) >= 3 * stage_bytes + 4096)
        each++;
    for (;; each--) {
        budget = 227 * 1024 / each - 1024 - 1024 - (uint32_t)sizeof(FewSmem);
        if (each == 1 || budget >= std::max(2 * stage_bytes, p.tokens * kFewRows * 4))
            break;
    }
    p.stages = std::min<uint32_t>(budget / stage_bytes, kFewMaxStages);
    p.sums_at = 0;
    if (p.splits > 1 && p.stages > 2 && sums + 2 * stage_bytes <= budget) {
        p.stages = std::min((budget - sums) / stage_bytes, p.stages);
        p.sums_at = p.stages * stage_bytes;
    }
    p.smem_bytes = p.sums_at ? p.sums_at + sums : std::max(p.stages * stage_bytes, std::max(sums, p.tokens * kFewRows * 4));
}

template <int DT, LinearForm FORM>
static int launch_few(const Product &w, uint32_t k_blocks, cudaStream_t s)
{
    constexpr uint32_t tile_cols = few_cols<FORM>;
    const uint64_t elem = elem_bytes(DT);
    FewParams p = {};
    p.m = w.m;
    p.n = w.n;
    p.k_blocks = k_blocks;
    const uint32_t tiles = ceil_div(w.n, tile_cols);
    plan_few(p, tiles, (uint32_t)num_sms());
    p.out = w.out;
    p.activation = w.activation;
    p.c = w.c[0];
    p.g = w.c[1];
    p.u = w.c[2];
    p.ldc = w.ldc;
    p.a_scale = w.a_scale;
    p.b_scale = w.b_scale;
    p.u_scale = w.u_scale;
    p.bias = w.bias;
    p.status = w.status;
    FewMaps maps = {};
    int rc = make_matrix_map(&maps.x, w.a.base, w.m, w.k * elem, w.a.ld * elem, p.tokens);
    for (int i = 0; i < (FORM == kGated ? 2 : 1) && rc == CLPK_OK; i++)
        rc = make_matrix_map(&maps.w[i], w.b[i].base, w.n, w.k * elem, w.b[i].ld * elem, tile_cols);
    if (rc != CLPK_OK)
        return rc;
    return launch_clusters(linear_few_kernel<DT, FORM>, "linear_few", tiles * p.splits, kFewThreads, p.smem_bytes + sizeof(FewSmem) + 1024, p.splits, s, maps, p);
}

// a product with few tokens or many
template <int DT, LinearForm FORM>
static int run_tokens(const Product &w, cudaStream_t s)
{
    const uint32_t k_blocks = linear_k_blocks(w.k, DT);
    if (few_tokens(w.m, ceil_div(w.n, few_cols<FORM>), k_blocks, (uint32_t)num_sms()))
        return launch_few<DT, FORM>(w, k_blocks, s);
    return launch_linear<DT, FORM>(w, k_blocks, s);
}

// ---- the backward pass: dg = dh * u * act'(g) and du = dh * act(g) ----------------------------------------
//
// Five arrays of 16-bit numbers pass by, ten bytes an element: bound by memory.  Eight elements a thread; 8192 x 8192 in 96 us, 7.0
// TB/s, and 125 behind products that have just written theirs.  The rounding of dg and du to 16 bits is what lets the tensor cores multiply them at full rate: it adds to
// the gradients an error of the size of their own rounding (bf16 0.0017 -> 0.0023 of the norm).
// Making them inside the products' launch, by warps that wait for a first tile, was built and measured: in a program that
// keeps the card at its power limit nothing is gained by overlap (1023 against 988 us at 8192 x 2048 x 8192).
struct GateParams {
    const void *dh, *g, *u;
    void *dg, *du;
    uint64_t ldh, ldw;                  // of the first three, and of the two in the workspace
    uint32_t m, f;
    uint32_t vectors;                   // of eight elements in a row
};

template <int DT>
__device__ __forceinline__ float2 widen(uint32_t w)
{
    if constexpr (DT == CLPK_DT_F16)
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// eight elements of a row of `f`, zeros beyond it
__device__ __forceinline__ uint4 load8(const void *base, uint64_t at, uint32_t left)
{
    const uint16_t *p = static_cast<const uint16_t *>(base) + at;
    if (left >= 8)
        return *reinterpret_cast<const uint4 *>(p);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
        if (i < left)
            w[i / 2] |= (uint32_t)p[i] << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT, int ACT>
__global__ void __launch_bounds__(256) gate_gradients_kernel(GateParams p)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / p.vectors;
    if (row >= p.m)
        return;
    const uint32_t col = (i - row * p.vectors) * 8, left = p.f - col;
    const uint64_t at = row * p.ldh + col;
    const uint4 vdh = load8(p.dh, at, left), vg = load8(p.g, at, left), vu = load8(p.u, at, left);
    const uint32_t dh[4] = {vdh.x, vdh.y, vdh.z, vdh.w}, g[4] = {vg.x, vg.y, vg.z, vg.w}, u[4] = {vu.x, vu.y, vu.z, vu.w};
    uint32_t dg[4], du[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 h2 = widen<DT>(dh[j]), g2 = widen<DT>(g[j]), u2 = widen<DT>(u[j]);
        float ax, dx, ay, dy;
        activate_both<ACT>(g2.x, ax, dx);
        activate_both<ACT>(g2.y, ay, dy);
        dg[j] = pack16(h2.x * u2.x * dx, h2.y * u2.y * dy, DT);
        du[j] = pack16(h2.x * ax, h2.y * ay, DT);
    }
    const uint64_t to = row * p.ldw + col;          // whole vectors: the workspace's pitch has room for them
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.dg) + to) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.du) + to) = make_uint4(du[0], du[1], du[2], du[3]);
}

template <int DT>
static int launch_gradients(const GateParams &p, int act, cudaStream_t s)
{
    const uint64_t vectors = (uint64_t)p.m * p.vectors;
    CLPK_REQUIRE(vectors <= (1ull << 32) - 256, "clpk_gated_ffn_backward: %u x %u is too large", p.m, p.f);
    const unsigned grid = (unsigned)((vectors + 255) / 256);
    switch (act) {
    case CLPK_ACT_SILU:      return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_SILU>, "gate_gradients", grid, 256, 0, s, p);
    case CLPK_ACT_GELU_TANH: return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_GELU_TANH>, "gate_gradients", grid, 256, 0, s, p);
    case CLPK_ACT_GELU:      return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_GELU>, "gate_gradients", grid, 256, 0, s, p);
    case CLPK_ACT_RELU:      return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_RELU>, "gate_gradients", grid, 256, 0, s, p);
    default:                 return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_SIGMOID>, "gate_gradients", grid, 256, 0, s, p);
    }
}

// elements from one row of dg or du to the next in the workspace
static uint64_t gradient_pitch(uint32_t f) { return ((uint64_t)f + 7) / 8 * 8; }

// Partial sums of K in the workspace -> the result.  Four columns per thread and step; 4 bytes an element and part, mostly from the
// L2 that they have just been written to.
struct JoinResult {
    const float *parts;                 // [parts][rows_all][cols_all]
    void *out;                          // [rows][cols], pitch ld
    uint64_t ld;
    uint32_t rows, rows_all, n_parts;
};
struct JoinParams {
    JoinResult r[3];
    uint32_t cols, cols_all;            // cols_all: a multiple of four
};

template <int DT>
__global__ void __launch_bounds__(128) join_parts_kernel(JoinParams p)
{
    griddep_wait();
    griddep_launch_dependents();
    const JoinResult &r = p.r[blockIdx.y];
    const uint32_t vectors = p.cols_all / 4;
    const uint64_t all = (uint64_t)r.rows * vectors, part = (uint64_t)r.rows_all * vectors;
    for (uint64_t i = (uint64_t)blockIdx.x * 128 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 128) {
        const float4 *from = reinterpret_cast<const float4 *>(r.parts) + i;
        float4 sum = *from;
#pragma unroll 8
        for (uint32_t k = 1; k < r.n_parts; k++) {
            const float4 v = from[k * part];
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        const uint64_t row = i / vectors;
        const uint32_t col = (uint32_t)(i - row * vectors) * 4;
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        few_store(r.out, DT, row * r.ld + col, p.cols - col, v);
    }
}

// What a tile counts for, in K blocks: a short sum takes as long as the tile before it takes to be stored, 1.5 us (tn = 128) to 2.1.
static uint32_t tile_blocks(const GradTiles &t) { return t.tiles ? std::max(ceil_div(t.blocks, t.parts), 7u) : 1; }

// The second tiles of the clusters that have one of the first more (a) and of the others (b), so that the longest cluster is about
// as short as it gets; returns its K blocks.
static uint64_t share_tiles(const GradTiles &first, const GradTiles &second, uint32_t clusters, uint32_t &share_a, uint32_t &share_b)
{
    const uint32_t more = first.tiles % clusters, each = first.tiles / clusters;
    const uint32_t fb = tile_blocks(first), sb = tile_blocks(second);
    // b - a is what one of the first is worth
    const uint64_t without = more ? (uint64_t)(clusters - more) * (fb / sb) : 0;
    const uint32_t about = second.tiles > without ? (uint32_t)((second.tiles - without) / clusters) : 0;
    uint64_t longest = ~0ull;
    for (uint32_t a = about ? about - 1 : 0; a <= about + 2; a++) {
        const uint32_t rest = (uint64_t)a * clusters < second.tiles ? second.tiles - a * clusters : 0;
        const uint32_t b = a + (rest ? ceil_div(rest, clusters - more) : 0);
        const uint64_t t = std::max(more ? (uint64_t)(each + 1) * fb + (uint64_t)a * sb : 0, (uint64_t)each * fb + (uint64_t)b * sb);
        if (t < longest) {
            longest = t;
            share_a = a;
            share_b = b;
        }
    }
    return longest;
}

constexpr uint32_t kGradPairs = 74;                         // of a whole B200: the workspace's size may not depend on the card at hand

// How the products of the backward pass are cut: tile width and parts of K, the cheapest by the estimate.  A set of tiles that fills
// the chip is whole, and so is one of the two (no shape gained more than 1 % by cutting both).  Over the 73 shapes that the
// estimate was fitted to this is 0.9 % slower than the fastest in the geometric mean, 9 % at most; over 73 others 1.7 %, where 59 are within
// 2 % and the worst takes 18.2 us uncut and 14.9 with dW in three parts (2467 x 919 x 138).  4103 x 170 x 3591 takes 71 us in tiles of 128
// columns, 58 in tiles of 256 and dx in two parts.
struct GradPlan {
    uint32_t tn, x_parts, w_parts;
};

static GradTiles x_tiles(uint32_t m, uint32_t d, uint32_t f, uint32_t tn, uint32_t parts)
{
    const uint32_t tiles_m = ceil_div(m, kLinearM);
    return {parts * tiles_m * ceil_div(d, tn), tiles_m, 2 * ceil_div(f, kLinearK), parts, 1};
}
static GradTiles w_tiles(uint32_t m, uint32_t d, uint32_t f, uint32_t tn, uint32_t parts)
{
    const uint32_t tiles_m = ceil_div(f, kLinearM);
    return {2 * parts * tiles_m * ceil_div(d, tn), tiles_m, ceil_div(m, kLinearK), parts, 2};
}

static uint64_t part_cols(uint32_t d) { return ((uint64_t)d + 3) / 4 * 4; }

// bytes of the fp32 results of all parts; none where K is whole
static uint64_t part_bytes(const GradTiles &t, uint32_t d) { return t.parts > 1 ? (uint64_t)t.products * t.parts * t.tiles_m * kLinearM * part_cols(d) * 4 : 0; }

static const GradTiles &longer(const GradTiles &x, const GradTiles &w)
{
    return w.tiles == 0 || (x.tiles > 0 && x.blocks / x.parts >= w.blocks / w.parts) ? x : w;
}

static GradPlan plan_backward(uint32_t m, uint32_t d, uint32_t f)
{
    GradPlan plan = {256, 1, 1};
    float best = 1e30f;
    for (uint32_t tn = 128; tn <= 256; tn += 128) {
        const GradTiles whole[2] = {x_tiles(m, d, f, tn, 1), w_tiles(m, d, f, tn, 1)};
        const auto look = [&](uint32_t x_parts, uint32_t w_parts) {
            const GradTiles x = x_tiles(m, d, f, tn, x_parts), w = w_tiles(m, d, f, tn, w_parts);
            const GradTiles &first = longer(x, w), &second = &first == &x ? w : x;
            const uint32_t clusters = std::min(x.tiles + w.tiles, kGradPairs);
            uint32_t a, b;
            float t = linear_estimate((float)share_tiles(first, second, clusters, a, b), (float)ceil_div(x.tiles + w.tiles, clusters), tn, 1);
            if (x_parts + w_parts > 2)      // a launch, and each part's sums written and read
                t += 2.0f + (float)(part_bytes(x, d) + part_bytes(w, d)) / 1.5e6f;
            if (t < best) {
                best = t;
                plan = {tn, x_parts, w_parts};
            }
        };
        look(1, 1);
        for (int which = 0; which < 2; which++)
            for (const uint32_t parts : {2, 3, 4, 6, 8, 12, 16, 24, 32})
                if (whole[which].tiles < kGradPairs && whole[which].blocks >= 8 * parts)
                    look(which ? 1 : parts, which ? parts : 1);
    }
    return plan;
}

// Sizes whose tiles and parts 32 bits can count: 2^25 of dx, and of dWg, are more than any card holds the results of.
static int check_backward_sizes(uint32_t m, uint32_t d, uint32_t f)
{
    const uint64_t cols = ((uint64_t)d + 127) / 128, x = ((uint64_t)m + kLinearM - 1) / kLinearM * cols, w = ((uint64_t)f + kLinearM - 1) / kLinearM * cols;
    CLPK_REQUIRE(m <= kMostRows && d <= kMostRows / 4 && f <= kMostRows / 4 && x <= 1u << 25 && w <= 1u << 25, "clpk_gated_ffn_backward: %u x %u x %u is too large", m, d, f);
    return CLPK_OK;
}

static uint64_t backward_bytes(uint32_t m, uint32_t d, uint32_t f, GradPlan &plan)
{
    const uint64_t gradients = 2 * (uint64_t)m * gradient_pitch(f) * 2;
    if (m == 0 || d == 0 || f == 0)
        return gradients;
    plan = plan_backward(m, d, f);
    return gradients + part_bytes(x_tiles(m, d, f, plan.tn, plan.x_parts), d) + part_bytes(w_tiles(m, d, f, plan.tn, plan.w_parts), d);
}

template <int DT>
static int run_backward(const clpk_gated_ffn_backward_args_t &a, const GradPlan &cut, cudaStream_t s)
{
    const uint64_t pitch = gradient_pitch(a.f);
    uint16_t *const dg = static_cast<uint16_t *>(a.d_workspace), *const du = dg + a.m * pitch;
    float *parts = reinterpret_cast<float *>(du + a.m * pitch);
    const GateParams gates = {a.d_dh, a.d_g, a.d_u, dg, du, a.ldh, pitch, a.m, a.f, (uint32_t)(pitch / 8)};
    int rc = launch_gradients<DT>(gates, a.activation, s);
    if (rc != CLPK_OK)
        return rc;

    const LinearPlan plan = {cut.tn, 1};
    GradTiles x = x_tiles(a.m, a.d, a.f, cut.tn, cut.x_parts), w = w_tiles(a.m, a.d, a.f, cut.tn, cut.w_parts);
    if (!a.d_dx)
        x.tiles = 0;
    if (!a.d_dwg)
        w.tiles = 0;
    GradParams p = {};
    p.segment = ceil_div(a.f, kLinearK);
    p.status = a.d_status;
    p.first = longer(x, w);
    p.second = &longer(x, w) == &x ? w : x;
    const uint32_t n_tiles = x.tiles + w.tiles;
    const uint32_t clusters = std::min(n_tiles, linear_resident(1)), tiles_n = ceil_div(a.d, cut.tn);
    share_tiles(p.first, p.second, clusters, p.share_a, p.share_b);
    p.first_each = p.first.tiles / clusters;
    p.first_more = p.first.tiles % clusters;
    for (GradTiles *set : {&p.first, &p.second}) {
        set->order = tile_order(set->tiles_m, tiles_n);
        set->by_product = divider(set->tiles_m * tiles_n);
        set->by_parts = divider(set->parts);
    }

    GradMaps maps = {};
    for (int i = 0; i < 2 && rc == CLPK_OK; i++) {
        const void *grad = i ? du : dg, *weight = i ? a.d_wu : a.d_wg;
        if (a.d_dx) {
            rc = make_matrix_map(&maps.dg[i], grad, a.m, (uint64_t)a.f * 2, pitch * 2, 128);
            if (rc == CLPK_OK)
                rc = make_matrix_map(&maps.w[i], weight, a.f, (uint64_t)a.d * 2, a.ldw * 2, kLinearK);
        }
        if (rc == CLPK_OK && a.d_dwg)
            rc = make_matrix_map(&maps.dg_t[i], grad, a.m, (uint64_t)a.f * 2, pitch * 2, kLinearK);
    }
    if (rc == CLPK_OK && a.d_dwg)
        rc = make_matrix_map(&maps.x, a.d_x, a.m, (uint64_t)a.d * 2, a.ldx * 2, kLinearK);
    JoinParams join = {};
    uint32_t results = 0;
    join.cols = a.d;
    join.cols_all = (uint32_t)part_cols(a.d);
    uint64_t joined = 0;                                    // vectors of the largest result
    void *const out[3] = {a.d_dx, a.d_dwg, a.d_dwu};
    for (int i = 0; i < 3 && rc == CLPK_OK; i++) {
        if (!out[i])
            continue;
        const GradTiles &set = i ? w : x;
        const uint32_t rows = i ? a.f : a.m, rows_all = set.tiles_m * kLinearM;
        const uint64_t ld = i ? a.ldw : a.ldx;
        if (set.parts > 1) {
            p.c[i] = linear_result(parts, join.cols_all, set.parts * rows_all, join.cols_all, CLPK_DT_F32);
            join.r[results++] = {parts, out[i], ld, rows, rows_all, set.parts};
            joined = std::max(joined, (uint64_t)rows * join.cols_all / 4);
            parts += (uint64_t)set.parts * rows_all * join.cols_all;
        } else {
            p.c[i] = linear_result(out[i], ld, rows, a.d, DT);
        }
        rc = make_result_map(&maps.c[i], p.c[i]);
    }
    if (rc != CLPK_OK)
        return rc;
    rc = launch_linear_tiles<DT, kGradients>(maps, p, plan, n_tiles, "linear (gradients)", s);
    if (rc != CLPK_OK || results == 0)
        return rc;
    const unsigned grid = (unsigned)std::min<uint64_t>((joined + 127) / 128, 16u * (uint32_t)num_sms());
    return launch_behind(join_parts_kernel<DT>, "join_parts", dim3(grid, results), 128, 0, s, join);
}

// ---- what the calls ask of their arguments ------------------------------------------------------------

// the pitch of a matrix with `cols` columns; 0 in *ld: rows one behind another
static int check_matrix(const char *what, const char *name, const void *base, uint64_t cols, uint64_t *ld, int dtype)
{
    const uint64_t elem = elem_bytes(dtype);
    if (*ld == 0)
        *ld = cols;
    CLPK_REQUIRE(base, "%s: %s is NULL", what, name);
    CLPK_REQUIRE(*ld >= cols, "%s: the pitch of %s, %llu, is shorter than its rows of %llu", what, name, (unsigned long long)*ld, (unsigned long long)cols);
    CLPK_REQUIRE(*ld < 1ull << 35, "%s: the pitch of %s, %llu, is too large", what, name, (unsigned long long)*ld);
    CLPK_REQUIRE(*ld * elem % 16 == 0 && (uintptr_t)base % 16 == 0, "%s: %s must start on 16 bytes and its pitch (%llu elements of %llu bytes) be a multiple of 16 bytes",
                 what, name, (unsigned long long)*ld, (unsigned long long)elem);
    return CLPK_OK;
}

#define CLPK_TRY(call)            \
    do {                          \
        const int rc__ = (call);  \
        if (rc__ != CLPK_OK)      \
            return rc__;          \
    } while (0)

static int check_status(const char *what, const uint32_t *status)
{
    CLPK_REQUIRE(status && (uintptr_t)status % 4 == 0, "%s: d_status must be a device word", what);
    return CLPK_OK;
}

static int check_scales(const char *what, const char *name, const float *scales)
{
    CLPK_REQUIRE(scales && (uintptr_t)scales % 4 == 0, "%s: %s must be an array of floats", what, name);
    return CLPK_OK;
}

constexpr uint32_t kMostI8 = 131071;                // products of magnitude 2^14 that a 32-bit sum holds

static int check_sizes(const char *what, uint32_t m, uint32_t n, uint32_t k, uint64_t elem)
{
    CLPK_REQUIRE(n > 0 && k > 0, "%s: only the number of tokens may be 0 (got %u x %u)", what, n, k);
    const uint64_t tiles = ((uint64_t)m + kLinearM - 1) / kLinearM * (((uint64_t)n + 31) / 32);           // at most
    CLPK_REQUIRE(m <= kMostRows && n * elem <= kMostRows && k * elem <= kMostRows && tiles <= 1u << 31, "%s: %u x %u x %u is too large", what, m, n, k);
    return CLPK_OK;
}

} // namespace clpk

using namespace clpk;

extern "C" {

int clpk_gemm_i8_scaled(const clpk_gemm_i8_scaled_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_gemm_i8_scaled";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_gemm_i8_scaled_args_t a = *args;
    CLPK_REQUIRE(a.out_dtype == CLPK_DT_F32 || a.out_dtype == CLPK_DT_F16 || a.out_dtype == CLPK_DT_BF16, "%s: out_dtype %d is not F32, F16 or BF16", what, a.out_dtype);
    CLPK_TRY(check_sizes(what, a.m, a.n, a.k, 4));
    CLPK_REQUIRE(a.k <= kMostI8, "%s: K = %u, and a 32-bit sum holds %u products", what, a.k, kMostI8);
    CLPK_TRY(check_status(what, a.d_status));
    cudaStream_t s = as_stream(stream);
    if (a.m == 0) {
        CLPK_CUDA(cudaMemsetAsync(a.d_status, 0, sizeof(uint32_t), s));
        return CLPK_OK;
    }
    CLPK_TRY(check_matrix(what, "d_a", a.d_a, a.k, &a.lda, CLPK_DT_I8));
    CLPK_TRY(check_matrix(what, "d_b", a.d_b, a.k, &a.ldb, CLPK_DT_I8));
    CLPK_TRY(check_matrix(what, "d_c", a.d_c, a.n, &a.ldc, a.out_dtype));
    CLPK_TRY(check_scales(what, "d_a_scale", a.d_a_scale));
    CLPK_TRY(check_scales(what, "d_b_scale", a.d_b_scale));
    CLPK_REQUIRE((uintptr_t)a.d_bias % elem_bytes(a.out_dtype) == 0, "%s: d_bias is not aligned to its elements", what);
    Product w = {};
    w.m = a.m;
    w.n = a.n;
    w.k = a.k;
    w.a = {a.d_a, a.lda};
    w.b[0] = {a.d_b, a.ldb};
    w.c[0] = a.d_c;
    w.ldc = a.ldc;
    w.out = a.out_dtype;
    w.a_scale = a.d_a_scale;
    w.b_scale = a.d_b_scale;
    w.bias = a.d_bias;
    w.status = a.d_status;
    return run_tokens<CLPK_DT_I8, kScaled>(w, s);
}

int clpk_gated_ffn(const clpk_gated_ffn_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_gated_ffn";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_gated_ffn_args_t a = *args;
    const bool i8 = a.dtype == CLPK_DT_I8;
    CLPK_REQUIRE(i8 || a.dtype == CLPK_DT_BF16 || a.dtype == CLPK_DT_F16, "%s: dtype %d is not BF16, F16 or I8", what, a.dtype);
    CLPK_REQUIRE(!i8 || a.out_dtype == CLPK_DT_F32 || a.out_dtype == CLPK_DT_F16 || a.out_dtype == CLPK_DT_BF16, "%s: out_dtype %d is not F32, F16 or BF16", what, a.out_dtype);
    CLPK_REQUIRE(a.activation >= 0 && a.activation < CLPK_ACT_COUNT, "%s: unknown activation %d", what, a.activation);
    CLPK_TRY(check_sizes(what, a.m, a.f, a.d, 4));
    CLPK_REQUIRE(!i8 || a.d <= kMostI8, "%s: d = %u, and a 32-bit sum holds %u products", what, a.d, kMostI8);
    CLPK_TRY(check_status(what, a.d_status));
    CLPK_REQUIRE((a.d_g != nullptr) == (a.d_u != nullptr), "%s: d_g and d_u: give both, or neither", what);
    CLPK_REQUIRE(!i8 || !a.d_g, "%s: g and u are not kept in 8 bits", what);
    cudaStream_t s = as_stream(stream);
    if (a.m == 0) {
        CLPK_CUDA(cudaMemsetAsync(a.d_status, 0, sizeof(uint32_t), s));
        return CLPK_OK;
    }
    const int out = i8 ? a.out_dtype : a.dtype;
    CLPK_TRY(check_matrix(what, "d_x", a.d_x, a.d, &a.ldx, a.dtype));
    CLPK_TRY(check_matrix(what, "d_wg", a.d_wg, a.d, &a.ldw, a.dtype));
    CLPK_TRY(check_matrix(what, "d_wu", a.d_wu, a.d, &a.ldw, a.dtype));
    CLPK_TRY(check_matrix(what, "d_h", a.d_h, a.f, &a.ldh, out));
    if (a.d_g) {
        CLPK_TRY(check_matrix(what, "d_g", a.d_g, a.f, &a.ldh, out));
        CLPK_TRY(check_matrix(what, "d_u", a.d_u, a.f, &a.ldh, out));
    }
    if (i8) {
        CLPK_TRY(check_scales(what, "d_x_scale", a.d_x_scale));
        CLPK_TRY(check_scales(what, "d_wg_scale", a.d_wg_scale));
        CLPK_TRY(check_scales(what, "d_wu_scale", a.d_wu_scale));
    }
    Product w = {};
    w.m = a.m;
    w.n = a.f;
    w.k = a.d;
    w.a = {a.d_x, a.ldx};
    w.b[0] = {a.d_wg, a.ldw};
    w.b[1] = {a.d_wu, a.ldw};
    w.c[0] = a.d_h;
    w.c[1] = a.d_g;
    w.c[2] = a.d_u;
    w.ldc = a.ldh;
    w.out = out;
    w.activation = a.activation;
    w.status = a.d_status;
    if (i8) {
        w.a_scale = a.d_x_scale;
        w.b_scale = a.d_wg_scale;
        w.u_scale = a.d_wu_scale;
        return run_tokens<CLPK_DT_I8, kGated>(w, s);
    }
    return a.dtype == CLPK_DT_F16 ? run_tokens<CLPK_DT_F16, kGated>(w, s) : run_tokens<CLPK_DT_BF16, kGated>(w, s);
}

int clpk_gated_ffn_backward_workspace_bytes(int dtype, uint32_t m, uint32_t d, uint32_t f, size_t *bytes)
{
    CLPK_REQUIRE(bytes, "bytes is NULL");
    *bytes = 0;
    CLPK_REQUIRE(dtype == CLPK_DT_BF16 || dtype == CLPK_DT_F16, "clpk_gated_ffn_backward: dtype %d is not BF16 or F16", dtype);
    CLPK_TRY(check_backward_sizes(m, d, f));
    GradPlan plan;
    *bytes = (size_t)backward_bytes(m, d, f, plan);
    return CLPK_OK;
}

int clpk_gated_ffn_backward(const clpk_gated_ffn_backward_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_gated_ffn_backward";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_gated_ffn_backward_args_t a = *args;
    CLPK_REQUIRE(a.dtype == CLPK_DT_BF16 || a.dtype == CLPK_DT_F16, "%s: dtype %d is not BF16 or F16", what, a.dtype);
    CLPK_TRY(check_backward_sizes(a.m, a.d, a.f));
    GradPlan cut = {};
    const size_t need = (size_t)backward_bytes(a.m, a.d, a.f, cut);
    CLPK_REQUIRE(a.activation >= 0 && a.activation < CLPK_ACT_COUNT, "%s: unknown activation %d", what, a.activation);
    CLPK_TRY(check_sizes(what, a.m, a.f, a.d, 4));
    CLPK_TRY(check_status(what, a.d_status));
    CLPK_REQUIRE((a.d_dwg != nullptr) == (a.d_dwu != nullptr), "%s: d_dwg and d_dwu: give both, or neither", what);
    if (a.d_dwg) {
        CLPK_TRY(check_matrix(what, "d_dwg", a.d_dwg, a.d, &a.ldw, a.dtype));
        CLPK_TRY(check_matrix(what, "d_dwu", a.d_dwu, a.d, &a.ldw, a.dtype));
    }
    cudaStream_t s = as_stream(stream);
    if (a.m == 0 || (!a.d_dx && !a.d_dwg)) {
        CLPK_CUDA(cudaMemsetAsync(a.d_status, 0, sizeof(uint32_t), s));
        for (void *w : {a.d_dwg, a.d_dwu})
            if (w)
                CLPK_CUDA(cudaMemset2DAsync(w, a.ldw * 2, 0, (size_t)a.d * 2, a.f, s));
        return CLPK_OK;
    }
    CLPK_TRY(check_matrix(what, "d_dh", a.d_dh, a.f, &a.ldh, a.dtype));
    CLPK_TRY(check_matrix(what, "d_g", a.d_g, a.f, &a.ldh, a.dtype));
    CLPK_TRY(check_matrix(what, "d_u", a.d_u, a.f, &a.ldh, a.dtype));
    CLPK_REQUIRE(a.d_workspace && a.workspace_bytes >= need && (uintptr_t)a.d_workspace % 16 == 0,
                 "%s: needs a 16-byte aligned workspace of %zu bytes", what, need);
    if (a.d_dx) {
        CLPK_TRY(check_matrix(what, "d_dx", a.d_dx, a.d, &a.ldx, a.dtype));
        CLPK_TRY(check_matrix(what, "d_wg", a.d_wg, a.d, &a.ldw, a.dtype));
        CLPK_TRY(check_matrix(what, "d_wu", a.d_wu, a.d, &a.ldw, a.dtype));
    }
    if (a.d_dwg)
        CLPK_TRY(check_matrix(what, "d_x", a.d_x, a.d, &a.ldx, a.dtype));

    return a.dtype == CLPK_DT_F16 ? run_backward<CLPK_DT_F16>(a, cut, s) : run_backward<CLPK_DT_BF16>(a, cut, s);
}

} // extern "C"
