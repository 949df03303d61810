// Layer norm and its gradients.
//
//   y = (x - mean) * rstd * w + b                     mean = sum x / d, rstd = 1 / sqrt(sum (x - mean)^2 / d + eps)
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) g = dy * w, xhat = (x - mean) * rstd
//   dw = sum over rows of dy * xhat, db = sum over rows of dy
//
// Bound by memory: x is read once and y written once, x and dy read and dx written once.  A row stays in the registers of the threads
// that share it, as the vectors it was loaded in, and the squares are summed about the mean: that is a second pass over registers,
// and it keeps the digits that sum x^2 - d mean^2 loses where the mean is large.
//
// dw and db are sums down the columns.  A CTA takes every gridDim-th row; a thread has the same columns of each, so that its share
// of both sums stays in registers, and one part for each CTA goes to the workspace, which a second kernel adds up: 8 bytes a column
// and CTA beside 6 a column and row.  The order of the sums depends on the sizes alone.
#include "../clpk_elements.cuh"
#include "../clpk_internal.h"
#include "../clpk_ptx.cuh"

#include <algorithm>

namespace clpk {

struct NormParams {
    const void *x, *weight, *bias;
    void *y;
    float *mean, *rstd;
    uint64_t ldx, ldy;
    uint32_t m, d;
    float eps;
};

// The sum over all threads of a row, the same in each.  `shared`: a word for each warp; not to be written again before all threads
// have come to the next barrier.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float *shared)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (THREADS > 32) {
        if ((threadIdx.x & 31) == 0)
            shared[threadIdx.x >> 5] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < THREADS / 32 ? shared[threadIdx.x & 31] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// Eight elements of a row, or as many as a vector has: what a thread loads at a time
template <int DT> constexpr int kPiece = Element<DT>::kPerVector;

// weights of a piece in fp32; `none` where there are none
template <int WDT, int N>
__device__ __forceinline__ void load_weights(float (&w)[N], const void *base, uint32_t at, uint32_t d, float none)
{
    if (!base) {
#pragma unroll
        for (int j = 0; j < N; j++)
            w[j] = none;
        return;
    }
    const typename Element<WDT>::T *p = static_cast<const typename Element<WDT>::T *>(base) + at;
    Raw<WDT, N> raw;
    if (at + N <= d)
        raw.load(p);
    else
        raw.load_some(p, at < d ? d - at : 0);
    raw.widen(w);
}

constexpr int kNormWarps = 4;                       // rows of a CTA whose rows are a warp's

// THREADS share a row of up to THREADS * ELEMS elements; rows and weights start on 16 bytes
template <int DT, int WDT, int THREADS, int ELEMS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kNormWarps : THREADS) layer_norm_kernel(NormParams p)
{
    using T = typename Element<DT>::T;
    constexpr int N = kPiece<DT>, kPieces = ELEMS / N;
    __shared__ float shared[2][THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = THREADS == 32 ? blockIdx.x * kNormWarps + (threadIdx.x >> 5) : blockIdx.x, t = threadIdx.x % THREADS;
    if (row >= p.m)                                 // whole warps, and THREADS == 32 alone: no barrier follows
        return;
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    Raw<DT, N> raw[kPieces];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const uint32_t at = (i * THREADS + t) * N;
        if (at + N <= p.d)
            raw[i].load(x + at);
        else
            raw[i].load_some(x + at, at < p.d ? p.d - at : 0);
    }
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        float v[N];
        raw[i].widen(v);
#pragma unroll
        for (int j = 0; j < N; j++)
            sum += v[j];
    }
    const float mean = row_sum<THREADS>(sum, shared[0]) / (float)p.d;
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const uint32_t at = (i * THREADS + t) * N;
        float v[N];
        raw[i].widen(v);
#pragma unroll
        for (int j = 0; j < N; j++)
            if (at + N <= p.d || at + j < p.d)
                squares = fmaf(v[j] - mean, v[j] - mean, squares);
    }
    const float rstd = 1.0f / sqrtf(row_sum<THREADS>(squares, shared[1]) / (float)p.d + p.eps);
    if (t == 0) {
        if (p.mean)
            p.mean[row] = mean;
        if (p.rstd)
            p.rstd[row] = rstd;
    }
    T *y = static_cast<T *>(p.y) + row * p.ldy;
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const uint32_t at = (i * THREADS + t) * N;
        if (at >= p.d)
            break;
        float v[N], w[N], b[N];
        raw[i].widen(v);
        load_weights<WDT>(w, p.weight, at, p.d, 1.0f);
        load_weights<WDT>(b, p.bias, at, p.d, 0.0f);
#pragma unroll
        for (int j = 0; j < N; j++)
            v[j] = fmaf((v[j] - mean) * rstd, w[j], b[j]);
        raw[i].round(v);
        if (at + N <= p.d)
            raw[i].store(y + at);
        else
            raw[i].store_some(y + at, p.d - at);
    }
}

// Rows that do not start on 16 bytes, or longer than the registers hold: element by element, read three times
template <int DT, int WDT>
__global__ void __launch_bounds__(256) layer_norm_plain_kernel(NormParams p)
{
    using E = Element<DT>;
    using W = Element<WDT>;
    __shared__ float shared[2][8];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = blockIdx.x;
    const typename E::T *x = static_cast<const typename E::T *>(p.x) + row * p.ldx;
    typename E::T *y = static_cast<typename E::T *>(p.y) + row * p.ldy;
    float sum = 0.0f, squares = 0.0f;
#pragma unroll 8
    for (uint64_t at = threadIdx.x; at < p.d; at += 256)
        sum += E::widen(x[at]);
    const float mean = row_sum<256>(sum, shared[0]) / (float)p.d;
#pragma unroll 8
    for (uint64_t at = threadIdx.x; at < p.d; at += 256) {
        const float off = E::widen(x[at]) - mean;
        squares = fmaf(off, off, squares);
    }
    const float rstd = 1.0f / sqrtf(row_sum<256>(squares, shared[1]) / (float)p.d + p.eps);
    if (threadIdx.x == 0) {
        if (p.mean)
            p.mean[row] = mean;
        if (p.rstd)
            p.rstd[row] = rstd;
    }
#pragma unroll 4
    for (uint64_t at = threadIdx.x; at < p.d; at += 256) {
        const float w = p.weight ? W::widen(static_cast<const typename W::T *>(p.weight)[at]) : 1.0f;
        const float b = p.bias ? W::widen(static_cast<const typename W::T *>(p.bias)[at]) : 0.0f;
        y[at] = E::round(fmaf((E::widen(x[at]) - mean) * rstd, w, b));
    }
}

// ---- gradients --------------------------------------------------------------------------------------------

struct NormGradParams {
    const void *x, *weight, *dy;
    const float *mean, *rstd;
    void *dx;
    float *parts;                                   // [gridDim][2][d]: shares of dw and db; NULL: not asked for
    uint64_t ldx, lddy, lddx;
    uint32_t m, d;
};

// both sums over all threads of a row; `shared` as in row_sum
template <int THREADS>
__device__ __forceinline__ float2 row_sums(float2 v, float2 *shared)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (THREADS > 32) {
        if ((threadIdx.x & 31) == 0)
            shared[threadIdx.x >> 5] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < THREADS / 32 ? shared[threadIdx.x & 31] : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int o = THREADS / 64; o > 0; o >>= 1) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        }
        v.x = __shfl_sync(0xffffffffu, v.x, 0);
        v.y = __shfl_sync(0xffffffffu, v.y, 0);
    }
    return v;
}

constexpr int kNormGradWarps = 8;                   // of a CTA whose rows are a warp's

template <int DT, int WDT, int THREADS, int ELEMS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kNormGradWarps : THREADS) layer_norm_gradients_kernel(NormGradParams p)
{
    using T = typename Element<DT>::T;
    constexpr int N = kPiece<DT>, kPieces = ELEMS / N, kRows = THREADS == 32 ? kNormGradWarps : 1;
    __shared__ float2 shared[2][THREADS / 32];
    __shared__ float joined[THREADS == 32 ? 2 * 32 * ELEMS : 1];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, t = threadIdx.x % THREADS;
    float dw[ELEMS] = {}, db[ELEMS] = {};
    uint32_t turn = 0;
    Raw<DT, N> x[kPieces], dy[kPieces];
    const uint32_t first = blockIdx.x * kRows + (kRows > 1 ? warp : 0), step = gridDim.x * kRows;
    auto ask = [&](uint32_t row) {                  // a row ahead, so that its way lies under the sums of the one before
        const T *from_x = static_cast<const T *>(p.x) + row * p.ldx, *from_dy = static_cast<const T *>(p.dy) + row * p.lddy;
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t at = (i * THREADS + t) * N;
            if (at + N <= p.d) {
                x[i].load(from_x + at);
                dy[i].load(from_dy + at);
            } else {
                x[i].load_some(from_x + at, at < p.d ? p.d - at : 0);
                dy[i].load_some(from_dy + at, at < p.d ? p.d - at : 0);
            }
        }
    };
    if (first < p.m)
        ask(first);
    for (uint64_t row = first; row < p.m; row += step) {
        const float mean = p.mean[row], rstd = p.rstd[row];
        float hat[ELEMS], g[ELEMS];
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t at = (i * THREADS + t) * N;
            float vx[N], vdy[N], w[N];
            x[i].widen(vx);
            dy[i].widen(vdy);
            load_weights<WDT>(w, p.weight, at, p.d, 1.0f);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int e = i * N + j;
                // behind the row x and dy are zeros, and a mean or rstd that is not finite must not come back in
                hat[e] = at + N <= p.d || at + j < p.d ? (vx[j] - mean) * rstd : 0.0f;
                g[e] = vdy[j] * w[j];
                dw[e] = fmaf(vdy[j], hat[e], dw[e]);
                db[e] += vdy[j];
                sum.x += g[e];
                sum.y = fmaf(g[e], hat[e], sum.y);
            }
        }
        if (row + step < p.m)
            ask((uint32_t)(row + step));
        if (!p.dx)
            continue;
        sum = row_sums<THREADS>(sum, shared[turn]);
        turn ^= 1;
        const float c1 = sum.x / (float)p.d, c2 = sum.y / (float)p.d;
        T *dx = static_cast<T *>(p.dx) + row * p.lddx;
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t at = (i * THREADS + t) * N;
            if (at >= p.d)
                break;
            float v[N];
#pragma unroll
            for (int j = 0; j < N; j++)
                v[j] = rstd * (g[i * N + j] - c1 - hat[i * N + j] * c2);
            Raw<DT, N> out;
            out.round(v);
            if (at + N <= p.d)
                out.store(dx + at);
            else
                out.store_some(dx + at, p.d - at);
        }
    }
    if (!p.parts)
        return;
    float *part = p.parts + (uint64_t)blockIdx.x * 2 * p.d;
    if constexpr (THREADS > 32) {
#pragma unroll
        for (int i = 0; i < kPieces; i++)
#pragma unroll
            for (int j = 0; j < N; j++) {
                const uint32_t at = (i * THREADS + t) * N + j;
                if (at < p.d) {
                    part[at] = dw[i * N + j];
                    part[p.d + at] = db[i * N + j];
                }
            }
    } else {
        // the warps' shares, one warp after another
        for (uint32_t w = 0; w < kNormGradWarps; w++) {
            if (w == warp) {
#pragma unroll
                for (int e = 0; e < ELEMS; e++) {
                    const uint32_t at = e * 32 + t;
                    joined[at] = w ? joined[at] + dw[e] : dw[e];
                    joined[32 * ELEMS + at] = w ? joined[32 * ELEMS + at] + db[e] : db[e];
                }
            }
            __syncthreads();
        }
        for (uint32_t e = warp; e < ELEMS; e += kNormGradWarps) {
            const uint32_t at = (e / N * 32 + t) * N + e % N;
            if (at < p.d) {
                part[at] = joined[e * 32 + t];
                part[p.d + at] = joined[32 * ELEMS + e * 32 + t];
            }
        }
    }
}

// Rows that do not start on 16 bytes, or are too long for registers: dx of a row by a CTA, element by element, read twice
template <int DT, int WDT>
__global__ void __launch_bounds__(256) layer_norm_plain_dx_kernel(NormGradParams p)
{
    using E = Element<DT>;
    using W = Element<WDT>;
    __shared__ float2 shared[8];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t row = blockIdx.x;
    const typename E::T *x = static_cast<const typename E::T *>(p.x) + row * p.ldx, *dy = static_cast<const typename E::T *>(p.dy) + row * p.lddy;
    typename E::T *dx = static_cast<typename E::T *>(p.dx) + row * p.lddx;
    const float mean = p.mean[row], rstd = p.rstd[row];
    auto values = [&](uint64_t at, float &hat, float &g) {
        hat = (E::widen(x[at]) - mean) * rstd;
        g = E::widen(dy[at]) * (p.weight ? W::widen(static_cast<const typename W::T *>(p.weight)[at]) : 1.0f);
    };
    float2 sum = make_float2(0.0f, 0.0f);
    float hat, g;
#pragma unroll 4
    for (uint64_t at = threadIdx.x; at < p.d; at += 256) {
        values(at, hat, g);
        sum.x += g;
        sum.y = fmaf(g, hat, sum.y);
    }
    sum = row_sums<256>(sum, shared);
    const float c1 = sum.x / (float)p.d, c2 = sum.y / (float)p.d;
#pragma unroll 4
    for (uint64_t at = threadIdx.x; at < p.d; at += 256) {
        values(at, hat, g);
        dx[at] = E::round(rstd * (g - c1 - hat * c2));
    }
}

// ... and their shares of dw and db: a thread has a column, gridDim.y CTAs share the rows
template <int DT>
__global__ void __launch_bounds__(256) layer_norm_plain_columns_kernel(NormGradParams p)
{
    using E = Element<DT>;
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t col = blockIdx.x * 256 + threadIdx.x;
    if (col >= p.d)
        return;
    float dw = 0.0f, db = 0.0f;
#pragma unroll 4
    for (uint64_t row = blockIdx.y; row < p.m; row += gridDim.y) {
        const float g = E::widen(static_cast<const typename E::T *>(p.dy)[row * p.lddy + col]);
        dw = fmaf(g, (E::widen(static_cast<const typename E::T *>(p.x)[row * p.ldx + col]) - p.mean[row]) * p.rstd[row], dw);
        db += g;
    }
    float *part = p.parts + (uint64_t)blockIdx.y * 2 * p.d;
    part[col] = dw;
    part[p.d + col] = db;
}

struct NormJoinParams {
    const float *parts;
    void *out[2];                                   // dw and db, either may be NULL
    uint32_t n_parts, d;
};

// The parts' sums, rounded: a lane has a column, the eight warps an eighth of the parts each
template <int WDT>
__global__ void __launch_bounds__(256) layer_norm_join_kernel(NormJoinParams p)
{
    __shared__ float sums[8][32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane, which = blockIdx.y;
    if (!p.out[which])
        return;
    float sum = 0.0f;
    if (col < p.d) {
        const float *from = p.parts + (uint64_t)which * p.d + col;
#pragma unroll 8
        for (uint32_t i = warp; i < p.n_parts; i += 8)
            sum += from[(uint64_t)i * 2 * p.d];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp > 0 || col >= p.d)
        return;
#pragma unroll
    for (uint32_t w = 1; w < 8; w++)
        sum += sums[w][lane];
    static_cast<typename Element<WDT>::T *>(p.out[which])[col] = Element<WDT>::round(sum);
}

// ---- host side ------------------------------------------------------------------------------------------

constexpr uint32_t kNormLongest = 32768, kNormGradLongest = 16384;      // elements of a row in registers

template <int DT, int WDT>
static int launch_norm(const NormParams &p, bool aligned, cudaStream_t s)
{
    if (!aligned || p.d > kNormLongest)
        return launch_behind(layer_norm_plain_kernel<DT, WDT>, "layer_norm_plain", p.m, 256, 0, s, p);
    const unsigned by_warps = (p.m - 1) / kNormWarps + 1;
    if (p.d <= 256)
        return launch_behind(layer_norm_kernel<DT, WDT, 32, 8>, "layer_norm", by_warps, 32 * kNormWarps, 0, s, p);
    if (p.d <= 512)
        return launch_behind(layer_norm_kernel<DT, WDT, 32, 16>, "layer_norm", by_warps, 32 * kNormWarps, 0, s, p);
    if (p.d <= 1024)
        return launch_behind(layer_norm_kernel<DT, WDT, 32, 32>, "layer_norm", by_warps, 32 * kNormWarps, 0, s, p);
    if (p.d <= 4096)
        return launch_behind(layer_norm_kernel<DT, WDT, 128, 32>, "layer_norm", p.m, 128, 0, s, p);
    if (p.d <= 8192)
        return launch_behind(layer_norm_kernel<DT, WDT, 256, 32>, "layer_norm", p.m, 256, 0, s, p);
    if (p.d <= 16384)
        return launch_behind(layer_norm_kernel<DT, WDT, 512, 32>, "layer_norm", p.m, 512, 0, s, p);
    return launch_behind(layer_norm_kernel<DT, WDT, 1024, 32>, "layer_norm", p.m, 1024, 0, s, p);
}

// Parts of dw and db: CTAs of layer_norm_gradients_kernel.  A whole B200's: the workspace's size may not depend on the card at hand.
static uint32_t norm_parts(uint32_t m, uint32_t d)
{
    constexpr uint32_t kSms = 148;
    if (d <= 1024)
        return std::min(m ? (m - 1) / kNormGradWarps + 1 : 1, 4 * kSms);
    return std::min(std::max(m, 1u), (d <= 2048 ? 4 : d <= 4096 ? 2 : 1) * kSms);
}

template <int DT, int WDT>
static int launch_norm_gradients(const NormGradParams &p, bool aligned, uint32_t parts, cudaStream_t s)
{
    if (!aligned || p.d > kNormGradLongest) {
        if (p.dx)
            CLPK_TRY(launch_behind(layer_norm_plain_dx_kernel<DT, WDT>, "layer_norm_plain_dx", p.m, 256, 0, s, p));
        return p.parts ? launch_behind(layer_norm_plain_columns_kernel<DT>, "layer_norm_plain_columns", dim3((p.d - 1) / 256 + 1, parts), 256, 0, s, p) : CLPK_OK;
    }
    if (p.d <= 256)
        return launch_behind(layer_norm_gradients_kernel<DT, WDT, 32, 8>, "layer_norm_gradients", parts, 32 * kNormGradWarps, 0, s, p);
    if (p.d <= 512)
        return launch_behind(layer_norm_gradients_kernel<DT, WDT, 32, 16>, "layer_norm_gradients", parts, 32 * kNormGradWarps, 0, s, p);
    if (p.d <= 1024)
        return launch_behind(layer_norm_gradients_kernel<DT, WDT, 32, 32>, "layer_norm_gradients", parts, 32 * kNormGradWarps, 0, s, p);
    if (p.d <= 2048)
        return launch_behind(layer_norm_gradients_kernel<DT, WDT, 128, 16>, "layer_norm_gradients", parts, 128, 0, s, p);
    if (p.d <= 4096)
        return launch_behind(layer_norm_gradients_kernel<DT, WDT, 256, 16>, "layer_norm_gradients", parts, 256, 0, s, p);
    if (p.d <= 8192)
        return launch_behind(layer_norm_gradients_kernel<DT, WDT, 512, 16>, "layer_norm_gradients", parts, 512, 0, s, p);
    return launch_behind(layer_norm_gradients_kernel<DT, WDT, 512, 32>, "layer_norm_gradients", parts, 512, 0, s, p);
}

// calls f<DT, WDT>
#define CLPK_BY_TYPES(dtype, weight_dtype, f, ...)                                                                            \
    ((dtype) == CLPK_DT_F32    ? f<CLPK_DT_F32, CLPK_DT_F32>(__VA_ARGS__)                                                     \
     : (dtype) == CLPK_DT_BF16 ? ((weight_dtype) == CLPK_DT_F32 ? f<CLPK_DT_BF16, CLPK_DT_F32>(__VA_ARGS__) : f<CLPK_DT_BF16, CLPK_DT_BF16>(__VA_ARGS__)) \
                               : ((weight_dtype) == CLPK_DT_F32 ? f<CLPK_DT_F16, CLPK_DT_F32>(__VA_ARGS__) : f<CLPK_DT_F16, CLPK_DT_F16>(__VA_ARGS__)))

static int check_norm(const char *what, int dtype, int weight_dtype, uint32_t m, uint32_t d)
{
    CLPK_REQUIRE(dtype == CLPK_DT_F32 || dtype == CLPK_DT_F16 || dtype == CLPK_DT_BF16, "%s: dtype %d is not F32, F16 or BF16", what, dtype);
    CLPK_REQUIRE(weight_dtype == dtype || weight_dtype == CLPK_DT_F32, "%s: weight_dtype %d is neither dtype nor F32", what, weight_dtype);
    CLPK_REQUIRE(d > 0, "%s: rows of no elements", what);
    CLPK_REQUIRE(m <= 0x7FFFFFFFu && d <= 1u << 30, "%s: %u x %u is too large", what, m, d);
    return CLPK_OK;
}

// the pitch of rows of d elements; 0 in *ld: one behind another.  Whether they all start on 16 bytes: *aligned stays.
static int check_rows(const char *what, const char *name, const void *base, uint32_t d, uint64_t *ld, int dtype, bool *aligned)
{
    const uint64_t elem = element_bytes(dtype);
    if (*ld == 0)
        *ld = d;
    CLPK_REQUIRE(base, "%s: %s is NULL", what, name);
    CLPK_REQUIRE(*ld >= d && *ld < 1ull << 35, "%s: the pitch of %s, %llu, is shorter than its rows of %u, or too large", what, name, (unsigned long long)*ld, d);
    CLPK_REQUIRE((uintptr_t)base % elem == 0, "%s: %s is not aligned to its elements", what, name);
    *aligned = *aligned && (uintptr_t)base % 16 == 0 && *ld * elem % 16 == 0;
    return CLPK_OK;
}

// an array that may be NULL
static int check_array(const char *what, const char *name, const void *base, int dtype, bool *aligned)
{
    CLPK_REQUIRE((uintptr_t)base % element_bytes(dtype) == 0, "%s: %s is not aligned to its elements", what, name);
    *aligned = *aligned && (uintptr_t)base % 16 == 0;
    return CLPK_OK;
}

static uint64_t norm_workspace(uint32_t m, uint32_t d)
{
    // fewer rows have no more parts
    return (uint64_t)norm_parts(m, d) * 2 * d * sizeof(float);
}

} // namespace clpk

using namespace clpk;

extern "C" {

int clpk_layer_norm(const clpk_layer_norm_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_layer_norm";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_layer_norm_args_t a = *args;
    CLPK_TRY(check_norm(what, a.dtype, a.weight_dtype, a.m, a.d));
    CLPK_REQUIRE(a.eps >= 0.0f && a.eps <= 3.4e38f, "%s: eps %g is not a number that is 0 or more", what, (double)a.eps);
    if (a.m == 0)
        return CLPK_OK;
    bool aligned = true, any = true;
    CLPK_TRY(check_rows(what, "d_x", a.d_x, a.d, &a.ldx, a.dtype, &aligned));
    CLPK_TRY(check_rows(what, "d_y", a.d_y, a.d, &a.ldy, a.dtype, &aligned));
    CLPK_TRY(check_array(what, "d_weight", a.d_weight, a.weight_dtype, &aligned));
    CLPK_TRY(check_array(what, "d_bias", a.d_bias, a.weight_dtype, &aligned));
    CLPK_TRY(check_array(what, "d_mean", a.d_mean, CLPK_DT_F32, &any));
    CLPK_TRY(check_array(what, "d_rstd", a.d_rstd, CLPK_DT_F32, &any));
    const NormParams p = {a.d_x, a.d_weight, a.d_bias, a.d_y, a.d_mean, a.d_rstd, a.ldx, a.ldy, a.m, a.d, a.eps};
    return CLPK_BY_TYPES(a.dtype, a.weight_dtype, launch_norm, p, aligned, as_stream(stream));
}

int clpk_layer_norm_backward_workspace_bytes(uint32_t m, uint32_t d, size_t *bytes)
{
    CLPK_REQUIRE(bytes, "bytes is NULL");
    *bytes = 0;
    CLPK_TRY(check_norm("clpk_layer_norm_backward", CLPK_DT_F32, CLPK_DT_F32, m, d));
    *bytes = (size_t)norm_workspace(m, d);
    return CLPK_OK;
}

int clpk_layer_norm_backward(const clpk_layer_norm_backward_args_t *args, void *stream)
{
    CLPK_TRY(require_sm100());
    const char *what = "clpk_layer_norm_backward";
    CLPK_REQUIRE(args, "%s: args is NULL", what);
    clpk_layer_norm_backward_args_t a = *args;
    CLPK_TRY(check_norm(what, a.dtype, a.weight_dtype, a.m, a.d));
    bool aligned = true, any = true;
    CLPK_TRY(check_array(what, "d_dweight", a.d_dweight, a.weight_dtype, &any));
    CLPK_TRY(check_array(what, "d_dbias", a.d_dbias, a.weight_dtype, &any));
    cudaStream_t s = as_stream(stream);
    if (a.m == 0) {
        for (void *w : {a.d_dweight, a.d_dbias})
            if (w)
                CLPK_CUDA(cudaMemsetAsync(w, 0, a.d * element_bytes(a.weight_dtype), s));
        return CLPK_OK;
    }
    const bool columns = a.d_dweight || a.d_dbias;
    if (!a.d_dx && !columns)
        return CLPK_OK;
    CLPK_TRY(check_rows(what, "d_x", a.d_x, a.d, &a.ldx, a.dtype, &aligned));
    CLPK_TRY(check_rows(what, "d_dy", a.d_dy, a.d, &a.lddy, a.dtype, &aligned));
    CLPK_TRY(check_array(what, "d_weight", a.d_weight, a.weight_dtype, &aligned));
    CLPK_REQUIRE(a.d_mean && a.d_rstd, "%s: d_mean or d_rstd is NULL", what);
    CLPK_TRY(check_array(what, "d_mean", a.d_mean, CLPK_DT_F32, &any));
    CLPK_TRY(check_array(what, "d_rstd", a.d_rstd, CLPK_DT_F32, &any));
    if (a.d_dx)
        CLPK_TRY(check_rows(what, "d_dx", a.d_dx, a.d, &a.lddx, a.dtype, &aligned));
    const uint32_t parts = norm_parts(a.m, a.d);
    const uint64_t need = norm_workspace(a.m, a.d);
    CLPK_REQUIRE(!columns || (a.d_workspace && a.workspace_bytes >= need && (uintptr_t)a.d_workspace % 16 == 0), "%s: needs a 16-byte aligned workspace of %llu bytes",
                 what, (unsigned long long)need);
    const NormGradParams p = {a.d_x, a.d_weight, a.d_dy, a.d_mean, a.d_rstd, a.d_dx, columns ? static_cast<float *>(a.d_workspace) : nullptr,
                              a.ldx, a.lddy, a.lddx, a.m, a.d};
    const int rc = CLPK_BY_TYPES(a.dtype, a.weight_dtype, launch_norm_gradients, p, aligned, parts, s);
    if (rc != CLPK_OK || !columns)
        return rc;
    const NormJoinParams join = {p.parts, {a.d_dweight, a.d_dbias}, parts, a.d};
    const dim3 grid((a.d - 1) / 32 + 1, 2);
    switch (a.weight_dtype) {
    case CLPK_DT_F32: return launch_behind(layer_norm_join_kernel<CLPK_DT_F32>, "layer_norm_join", grid, 256, 0, s, join);
    case CLPK_DT_F16: return launch_behind(layer_norm_join_kernel<CLPK_DT_F16>, "layer_norm_join", grid, 256, 0, s, join);
    default:          return launch_behind(layer_norm_join_kernel<CLPK_DT_BF16>, "layer_norm_join", grid, 256, 0, s, join);
    }
}

} // extern "C"
