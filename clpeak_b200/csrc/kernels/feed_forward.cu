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

// ---- dg = dh * u * act'(g) and du = dh * act(g) -----------------------------------------------------------
//
// Five arrays of 16-bit numbers pass by, ten bytes an element: bound by memory.  Eight elements per step and thread.
struct GradParams {
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
__global__ void __launch_bounds__(256) gate_gradients_kernel(GradParams p)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint64_t all = (uint64_t)p.m * p.vectors;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / p.vectors;
        const uint32_t col = (uint32_t)(i - row * p.vectors) * 8, left = p.f - col;
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
}

template <int DT>
static int launch_gradients(const GradParams &p, int act, cudaStream_t s)
{
    const uint64_t blocks = ((uint64_t)p.m * p.vectors + 255) / 256;
    const unsigned grid = (unsigned)std::min<uint64_t>(blocks, 1u << 30);
    switch (act) {
    case CLPK_ACT_SILU:      return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_SILU>, "gate_gradients", grid, 256, 0, s, p);
    case CLPK_ACT_GELU_TANH: return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_GELU_TANH>, "gate_gradients", grid, 256, 0, s, p);
    case CLPK_ACT_GELU:      return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_GELU>, "gate_gradients", grid, 256, 0, s, p);
    case CLPK_ACT_RELU:      return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_RELU>, "gate_gradients", grid, 256, 0, s, p);
    default:                 return launch_behind(gate_gradients_kernel<DT, CLPK_ACT_SIGMOID>, "gate_gradients", grid, 256, 0, s, p);
    }
}

// ---- the products -------------------------------------------------------------------------------------------

struct Matrix {
    const void *base;
    uint64_t ld;                        // elements
};

// One product of a layer: sums over `k` of an m x n result.
struct Product {
    uint32_t m, n, k;
    Matrix a[2], b[2];                  // kGated: b[0] = Wg, b[1] = Wu
    int segments, products;             // pairs of operands that are added; products of the same shape
    void *c[3];                         // of each product; kGated: h, g, u
    uint64_t ldc;
    int out, activation;
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
    uint32_t *status;
};

struct LinearPlan {
    uint32_t tn, splits;
};

static uint64_t elem_bytes(int dtype) { return dtype == CLPK_DT_F32 ? 4 : dtype == CLPK_DT_I8 ? 1 : 2; }

// K blocks of 128 bytes (64 of 16-bit elements, whichever way they lie)
static uint32_t linear_k_blocks(const Product &w, int dtype) { return (uint32_t)(((uint64_t)w.k * elem_bytes(dtype) + kRowBytesK - 1) / kRowBytesK); }

static LinearPlan plan_linear(const Product &w, LinearForm form, uint32_t k_blocks, bool b_mn)
{
    const uint32_t pairs = (uint32_t)num_sms() / 2, cols = form == kGated ? 2 * w.n : w.n;
    LinearPlan plan = {256, 1};
    float best = 1e30f;
    for (uint32_t splits = 1; splits <= 4 && splits <= k_blocks; splits *= 2)
        for (uint32_t tn = b_mn ? 128 : 64; tn <= 256; tn += b_mn ? 128 : 64) {
            const uint32_t resident = splits == 1 ? pairs : splits == 2 ? pairs * 33 / 74 : pairs * 15 / 74;
            const uint64_t tiles = (uint64_t)w.products * ((w.m - 1) / kLinearM + 1) * ((cols - 1) / tn + 1);
            if (resident == 0)
                continue;
            const float waves = (float)((tiles - 1) / resident + 1), wide = (float)tn / 256.0f;
            float t = 3.9f + waves * ((float)((k_blocks - 1) / splits + 1) * (0.118f + 0.265f * wide) + 1.2f * wide);
            if (splits > 1)
                t += waves * (1.0f + 4.3f * wide);
            if (t < best) {
                best = t;
                plan = {tn, splits};
            }
        }
    return plan;
}

template <int DT, LinearForm FORM, bool kAMn, bool kBMn>
static int launch_linear(const Product &w, LinearPlan plan, uint32_t k_blocks, cudaStream_t s)
{
    const uint64_t elem = elem_bytes(DT);
    LinearMaps maps = {};
    int rc = CLPK_OK;
    for (int i = 0; i < 2; i++) {
        if (w.a[i].base) {
            rc = kAMn ? make_matrix_map(&maps.a[i], w.a[i].base, w.k, w.m * elem, w.a[i].ld * elem, 64)
                      : make_matrix_map(&maps.a[i], w.a[i].base, w.m, w.k * elem, w.a[i].ld * elem, 128);
            if (rc != CLPK_OK)
                return rc;
        }
        if (w.b[i].base) {
            rc = kBMn ? make_matrix_map(&maps.b[i], w.b[i].base, w.k, w.n * elem, w.b[i].ld * elem, 64)
                      : make_matrix_map(&maps.b[i], w.b[i].base, w.n, w.k * elem, w.b[i].ld * elem, plan.tn / 2);
            if (rc != CLPK_OK)
                return rc;
        }
    }
    for (int i = 0; i < 3; i++)
        if (w.c[i]) {
            rc = make_result_map(&maps.c[i], w.c[i], w.m, w.n, w.ldc, w.out);
            if (rc != CLPK_OK)
                return rc;
        }
    LinearParams p = {};
    p.m = w.m;
    p.n = w.n;
    p.products = (uint32_t)w.products;
    p.tiles_m = (w.m - 1) / kLinearM + 1;
    const uint32_t tile_cols = FORM == kGated ? plan.tn / 2 : plan.tn;
    p.tiles_n = (w.n - 1) / tile_cols + 1;
    p.group = 8;
    p.k_segment = k_blocks;
    p.k_blocks = k_blocks * (uint32_t)w.segments;
    p.tn = plan.tn;
    p.splits = plan.splits;
    p.out = w.out;
    p.activation = w.activation;
    p.keep = FORM == kGated && w.c[1] ? 1 : 0;
    p.ragged = w.n * elem_bytes(w.out) % 16 != 0;
    std::copy(w.c, w.c + 3, p.c);
    p.ldc = w.ldc;
    p.a_scale = w.a_scale;
    p.b_scale = w.b_scale;
    p.u_scale = w.u_scale;
    p.bias = w.bias;
    p.status = w.status;
    const uint32_t n_tiles = p.products * p.tiles_m * p.tiles_n, pairs = (uint32_t)num_sms() / 2;
    const uint32_t clusters = plan.splits > 1 ? n_tiles : std::min(n_tiles, pairs);
    constexpr size_t fixed = kEpilogueWarps * kStagingBytes + sizeof(LinearSmem) + 1024;
    p.kps = plan.tn <= 128 ? 2 : 1;
    const uint32_t stage_bytes = p.kps * linear_block_bytes(plan.tn);
    p.stages = std::min<uint32_t>((uint32_t)((kSmemMax - fixed) / stage_bytes), kLinearMaxStages);
    p.tmem_cols = 32;
    while (p.tmem_cols < (n_tiles > clusters ? 2 : 1) * plan.tn)
        p.tmem_cols *= 2;
    return launch_clusters(linear_kernel<DT, FORM, kAMn, kBMn>, "linear", clusters * 2 * plan.splits, kLinearThreads,
                           p.stages * stage_bytes + fixed, 2 * plan.splits, s, maps, p);
}

template <LinearForm FORM> constexpr uint32_t few_cols = FORM == kGated ? 64 : 128;      // features of a tile

// K ranges of linear_few_kernel: as many as the chip holds CTAs for at once, as long as each has some blocks of K; with long sums
// also where that loads the SMs more evenly.  Of 160 shapes (1 to 128 tokens) it is 1 % slower than the fastest in the geometric
// mean.  What it decides: int8 1 x 4096 x 4096 in one range 9.2 us, in four 5.2; 8 x 30080 x 4096 (235 tiles) 26.7, in two 22.8.
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

template <int DT, LinearForm FORM>
static int launch_few(const Product &w, uint32_t k_blocks, cudaStream_t s)
{
    constexpr uint32_t tile_cols = few_cols<FORM>;
    const uint64_t elem = elem_bytes(DT);
    FewParams p = {};
    p.m = w.m;
    p.n = w.n;
    p.k_blocks = k_blocks;
    p.tokens = (w.m + 15) / 16 * 16;
    p.tmem_cols = 32;
    while (p.tmem_cols < p.tokens)
        p.tmem_cols *= 2;
    const uint32_t tiles = (w.n - 1) / tile_cols + 1, sms = (uint32_t)num_sms();
    p.splits = few_splits(w.m, tiles, k_blocks, sms);
    // as many CTAs as an SM gets share its memory; a ring has two stages at least, and is as large as the sums
    const uint32_t stage_bytes = kHalfTileBytes + p.tokens * kRowBytesK, sums = p.splits * ((p.m + p.splits - 1) / p.splits) * kFewRows * 4;
    uint32_t each = std::min((tiles * p.splits - 1) / sms + 1, (uint32_t)kFewResident), budget = 0;
    if ((each == 2 || (each == 1 && k_blocks < 32 * p.splits)) && 227 * 1024 / (each + 1) >= 3 * stage_bytes + 4096)
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
    int rc = make_matrix_map(&maps.x, w.a[0].base, w.m, w.k * elem, w.a[0].ld * elem, p.tokens);
    for (int i = 0; i < (FORM == kGated ? 2 : 1) && rc == CLPK_OK; i++)
        rc = make_matrix_map(&maps.w[i], w.b[i].base, w.n, w.k * elem, w.b[i].ld * elem, tile_cols);
    if (rc != CLPK_OK)
        return rc;
    return launch_clusters(linear_few_kernel<DT, FORM>, "linear_few", tiles * p.splits, kFewThreads, p.smem_bytes + sizeof(FewSmem) + 1024, p.splits, s, maps, p);
}

// a product whose operands are contiguous along K, with few tokens or many
template <int DT, LinearForm FORM>
static int run_tokens(const Product &w, cudaStream_t s)
{
    const uint32_t k_blocks = linear_k_blocks(w, DT);
    if (few_tokens(w.m, (w.n - 1) / few_cols<FORM> + 1, k_blocks, (uint32_t)num_sms()))
        return launch_few<DT, FORM>(w, k_blocks, s);
    return launch_linear<DT, FORM, false, false>(w, plan_linear(w, FORM, k_blocks, false), k_blocks, s);
}

// a product of the backward pass: B contiguous along N, A along K or M
template <int DT, bool kAMn>
static int run_gradient(const Product &w, cudaStream_t s)
{
    const uint32_t k_blocks = linear_k_blocks(w, DT);
    return launch_linear<DT, kPlain, kAMn, true>(w, plan_linear(w, kPlain, k_blocks * (uint32_t)w.segments, true), k_blocks, s);
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
constexpr uint32_t kMostRows = 0x7FFFFF00u;         // coordinates of whole tiles are signed 32-bit numbers

static int check_sizes(const char *what, uint32_t m, uint32_t n, uint32_t k, uint64_t elem)
{
    CLPK_REQUIRE(n > 0 && k > 0, "%s: only the number of tokens may be 0 (got %u x %u)", what, n, k);
    CLPK_REQUIRE(m <= kMostRows && n * elem <= kMostRows && k * elem <= kMostRows, "%s: %u x %u x %u is too large", what, m, n, k);
    return CLPK_OK;
}

// bytes of one of the two gradients that the workspace holds
static uint64_t gradient_pitch(uint32_t f) { return ((uint64_t)f + 7) / 8 * 8; }

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
    w.a[0] = {a.d_a, a.lda};
    w.b[0] = {a.d_b, a.ldb};
    w.segments = w.products = 1;
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
    w.a[0] = {a.d_x, a.ldx};
    w.b[0] = {a.d_wg, a.ldw};
    w.b[1] = {a.d_wu, a.ldw};
    w.segments = w.products = 1;
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
    (void)d;
    *bytes = 2 * (size_t)m * gradient_pitch(f) * 2;
    return CLPK_OK;
}

int clpk_gated_ffn_backward(const clpk_gated_ffn_backward_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_gated_ffn_backward";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_gated_ffn_backward_args_t a = *args;
    size_t need = 0;
    CLPK_TRY(clpk_gated_ffn_backward_workspace_bytes(a.dtype, a.m, a.d, a.f, &need));
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

    const uint64_t ld = gradient_pitch(a.f);
    uint8_t *dg = static_cast<uint8_t *>(a.d_workspace), *du = dg + a.m * ld * 2;
    const GradParams gp = {a.d_dh, a.d_g, a.d_u, dg, du, a.ldh, ld, a.m, a.f, (uint32_t)(ld / 8)};
    CLPK_TRY(a.dtype == CLPK_DT_F16 ? launch_gradients<CLPK_DT_F16>(gp, a.activation, s) : launch_gradients<CLPK_DT_BF16>(gp, a.activation, s));
    if (a.d_dx) {
        Product w = {};
        w.m = a.m;
        w.n = a.d;
        w.k = a.f;
        w.a[0] = {dg, ld};
        w.a[1] = {du, ld};
        w.b[0] = {a.d_wg, a.ldw};
        w.b[1] = {a.d_wu, a.ldw};
        w.segments = 2;
        w.products = 1;
        w.c[0] = a.d_dx;
        w.ldc = a.ldx;
        w.out = a.dtype;
        w.status = a.d_status;
        CLPK_TRY((a.dtype == CLPK_DT_F16 ? run_gradient<CLPK_DT_F16, false>(w, s) : run_gradient<CLPK_DT_BF16, false>(w, s)));
    }
    if (a.d_dwg) {
        Product w = {};
        w.m = a.f;
        w.n = a.d;
        w.k = a.m;
        w.a[0] = {dg, ld};
        w.a[1] = {du, ld};
        w.b[0] = {a.d_x, a.ldx};
        w.segments = 1;
        w.products = 2;
        w.c[0] = a.d_dwg;
        w.c[1] = a.d_dwu;
        w.ldc = a.ldw;
        w.out = a.dtype;
        w.status = a.d_status;
        CLPK_TRY((a.dtype == CLPK_DT_F16 ? run_gradient<CLPK_DT_F16, true>(w, s) : run_gradient<CLPK_DT_BF16, true>(w, s)));
    }
    return CLPK_OK;
}

} // extern "C"
