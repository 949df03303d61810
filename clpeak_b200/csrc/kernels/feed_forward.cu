// The products of a gated feed-forward layer: both projections with the activation, their gradients, and products of 8-bit
// integers with scales for each token and channel.
//
//   forward    g = x Wg^T, u = x Wu^T, h = act(g) * u
//   backward   dg = dh * u * act'(g), du = dh * act(g);  dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//   8 bits     c = float(sum of int8 products) * a_scale * b_scale + bias, and the forward pass with such sums
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../clpk_activation.cuh"
#include "../clpk_internal.h"
#include "../clpk_ptx.cuh"

namespace clpk {

// a matrix whose element (i, k) lies at base[i * rows + k * cols]
struct Strided {
    const void *base;
    uint64_t rows, cols;
};

struct ProductParams {
    Strided a[2], b[2];
    uint32_t m, n, k;
    int segments;                       // products that are added: a[0] b[0]^T + a[1] b[1]^T
    int activation;
    void *c, *g, *u;
    uint64_t ldc;
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
};

template <typename T> __device__ __forceinline__ float to_float(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float activate_by(int act, float g)
{
    switch (act) {
    case CLPK_ACT_SILU:      return activate<CLPK_ACT_SILU>(g);
    case CLPK_ACT_GELU_TANH: return activate<CLPK_ACT_GELU_TANH>(g);
    case CLPK_ACT_GELU:      return activate<CLPK_ACT_GELU>(g);
    case CLPK_ACT_RELU:      return activate<CLPK_ACT_RELU>(g);
    default:                 return activate<CLPK_ACT_SIGMOID>(g);
    }
}

// 32 x 32 results a block, a thread four of a column, through 32 x 32 tiles in shared memory
template <typename T, typename Acc, typename Out, bool kGated>
__global__ void __launch_bounds__(256) product_kernel(ProductParams p)
{
    __shared__ Acc ta[32][33], tb[2][32][33];
    const uint32_t tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const uint32_t row0 = blockIdx.y * 32, col0 = blockIdx.x * 32;
    Acc acc[2][4] = {};
    griddep_wait();
    griddep_launch_dependents();
    for (int s = 0; s < p.segments; s++) {
        const Strided &a = p.a[s];
        for (uint32_t k0 = 0; k0 < p.k; k0 += 32) {
            for (uint32_t i = ty; i < 32; i += 8) {
                const uint32_t k = k0 + tx;
                ta[i][tx] = row0 + i < p.m && k < p.k ? (Acc)static_cast<const T *>(a.base)[(row0 + i) * a.rows + k * a.cols] : Acc(0);
                for (int o = 0; o < (kGated ? 2 : 1); o++) {
                    const Strided &b = p.b[kGated ? o : s];
                    tb[o][i][tx] = col0 + i < p.n && k < p.k ? (Acc)static_cast<const T *>(b.base)[(col0 + i) * b.rows + k * b.cols] : Acc(0);
                }
            }
            __syncthreads();
            for (uint32_t k = 0; k < 32; k++)
                for (uint32_t i = 0; i < 4; i++) {
                    acc[0][i] += ta[ty + 8 * i][k] * tb[0][tx][k];
                    if (kGated)
                        acc[1][i] += ta[ty + 8 * i][k] * tb[1][tx][k];
                }
            __syncthreads();
        }
    }
    const uint32_t col = col0 + tx;
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t row = row0 + ty + 8 * i;
        if (row >= p.m || col >= p.n)
            continue;
        const uint64_t at = row * p.ldc + col;
        float v = (float)acc[0][i];
        if (p.a_scale)
            v = v * p.a_scale[row] * p.b_scale[col];
        if constexpr (kGated) {
            float u = (float)acc[1][i];
            if (p.a_scale)
                u = u * p.a_scale[row] * p.u_scale[col];
            if (p.g) {
                static_cast<Out *>(p.g)[at] = from_float<Out>(v);
                static_cast<Out *>(p.u)[at] = from_float<Out>(u);
            }
            v = activate_by(p.activation, v) * u;
        } else if (p.bias) {
            v += to_float(static_cast<const Out *>(p.bias)[col]);
        }
        static_cast<Out *>(p.c)[at] = from_float<Out>(v);
    }
}

struct GradParams {
    const void *dh, *g, *u;
    void *dg, *du;
    uint64_t ldh, ldw;                  // of the first three, and of the two in the workspace
    uint32_t m, f;
};

template <typename T, int ACT>
__global__ void __launch_bounds__(256) gate_gradients_kernel(GradParams p)
{
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t col = blockIdx.x * 256 + threadIdx.x;
    if (col >= p.f)
        return;
    for (uint32_t row = blockIdx.y; row < p.m; row += gridDim.y) {
        const uint64_t at = row * p.ldh + col, to = row * p.ldw + col;
        const float dh = to_float(static_cast<const T *>(p.dh)[at]), u = to_float(static_cast<const T *>(p.u)[at]);
        float a, da;
        activate_both<ACT>(to_float(static_cast<const T *>(p.g)[at]), a, da);
        static_cast<T *>(p.dg)[to] = from_float<T>(dh * u * da);
        static_cast<T *>(p.du)[to] = from_float<T>(dh * a);
    }
}

template <typename T, typename Acc, typename Out, bool kGated>
static int launch_product(const ProductParams &p, uint32_t *status, cudaStream_t s)
{
    CLPK_CUDA(cudaMemsetAsync(status, 0, sizeof(uint32_t), s));
    product_kernel<T, Acc, Out, kGated><<<dim3((p.n + 31) / 32, (p.m + 31) / 32), 256, 0, s>>>(p);
    CLPK_LAUNCH_CHECK("product");
    return CLPK_OK;
}

template <bool kGated>
static int launch_i8(const ProductParams &p, int out_dtype, uint32_t *status, cudaStream_t s)
{
    switch (out_dtype) {
    case CLPK_DT_F32: return launch_product<int8_t, int32_t, float, kGated>(p, status, s);
    case CLPK_DT_F16: return launch_product<int8_t, int32_t, __half, kGated>(p, status, s);
    default:          return launch_product<int8_t, int32_t, __nv_bfloat16, kGated>(p, status, s);
    }
}

template <bool kGated>
static int launch_16(const ProductParams &p, int dtype, uint32_t *status, cudaStream_t s)
{
    return dtype == CLPK_DT_F16 ? launch_product<__half, float, __half, kGated>(p, status, s)
                                : launch_product<__nv_bfloat16, float, __nv_bfloat16, kGated>(p, status, s);
}

template <typename T>
static int launch_gradients(const GradParams &p, int act, cudaStream_t s)
{
    const dim3 grid((p.f + 255) / 256, std::min(p.m, 65535u));
    switch (act) {
    case CLPK_ACT_SILU:      gate_gradients_kernel<T, CLPK_ACT_SILU><<<grid, 256, 0, s>>>(p); break;
    case CLPK_ACT_GELU_TANH: gate_gradients_kernel<T, CLPK_ACT_GELU_TANH><<<grid, 256, 0, s>>>(p); break;
    case CLPK_ACT_GELU:      gate_gradients_kernel<T, CLPK_ACT_GELU><<<grid, 256, 0, s>>>(p); break;
    case CLPK_ACT_RELU:      gate_gradients_kernel<T, CLPK_ACT_RELU><<<grid, 256, 0, s>>>(p); break;
    default:                 gate_gradients_kernel<T, CLPK_ACT_SIGMOID><<<grid, 256, 0, s>>>(p); break;
    }
    CLPK_LAUNCH_CHECK("gate_gradients");
    return CLPK_OK;
}

// ---- what the calls ask of their arguments ------------------------------------------------------------

static uint64_t elem_bytes(int dtype) { return dtype == CLPK_DT_F32 ? 4 : dtype == CLPK_DT_I8 ? 1 : 2; }

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
    ProductParams p = {};
    p.a[0] = {a.d_a, a.lda, 1};
    p.b[0] = {a.d_b, a.ldb, 1};
    p.m = a.m;
    p.n = a.n;
    p.k = a.k;
    p.segments = 1;
    p.c = a.d_c;
    p.ldc = a.ldc;
    p.a_scale = a.d_a_scale;
    p.b_scale = a.d_b_scale;
    p.bias = a.d_bias;
    return launch_i8<false>(p, a.out_dtype, a.d_status, s);
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
    ProductParams p = {};
    p.a[0] = {a.d_x, a.ldx, 1};
    p.b[0] = {a.d_wg, a.ldw, 1};
    p.b[1] = {a.d_wu, a.ldw, 1};
    p.m = a.m;
    p.n = a.f;
    p.k = a.d;
    p.segments = 1;
    p.activation = a.activation;
    p.c = a.d_h;
    p.g = a.d_g;
    p.u = a.d_u;
    p.ldc = a.ldh;
    if (i8) {
        p.a_scale = a.d_x_scale;
        p.b_scale = a.d_wg_scale;
        p.u_scale = a.d_wu_scale;
        return launch_i8<true>(p, out, a.d_status, s);
    }
    return launch_16<true>(p, out, a.d_status, s);
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
    const GradParams gp = {a.d_dh, a.d_g, a.d_u, dg, du, a.ldh, ld, a.m, a.f};
    CLPK_TRY(a.dtype == CLPK_DT_F16 ? launch_gradients<__half>(gp, a.activation, s) : launch_gradients<__nv_bfloat16>(gp, a.activation, s));
    ProductParams p = {};
    if (a.d_dx) {
        p.a[0] = {dg, ld, 1};
        p.a[1] = {du, ld, 1};
        p.b[0] = {a.d_wg, 1, a.ldw};
        p.b[1] = {a.d_wu, 1, a.ldw};
        p.m = a.m;
        p.n = a.d;
        p.k = a.f;
        p.segments = 2;
        p.c = a.d_dx;
        p.ldc = a.ldx;
        CLPK_TRY(launch_16<false>(p, a.dtype, a.d_status, s));
    }
    for (int o = 0; o < 2 && a.d_dwg; o++) {
        p.a[0] = {o ? du : dg, 1, ld};
        p.b[0] = {a.d_x, 1, a.ldx};
        p.m = a.f;
        p.n = a.d;
        p.k = a.m;
        p.segments = 1;
        p.c = o ? a.d_dwu : a.d_dwg;
        p.ldc = a.ldw;
        CLPK_TRY(launch_16<false>(p, a.dtype, a.d_status, s));
    }
    return CLPK_OK;
}

} // extern "C"
