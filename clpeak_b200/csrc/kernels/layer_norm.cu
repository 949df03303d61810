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
// CTAs stay, with the weights in registers, and take every gridDim-th row; a thread copies its pieces of the rows that come next into
// shared memory of its own (cp.async) while it computes, so that an SM has 40 to 200 KB on their way whatever its threads wait for.
// 16384 x 8192 bf16: 90 to 96 us, 5.6 to 6.0 TB/s, 85 to 91 % of a copy's rate (149 without rows ahead); what is missing is the wait for
// a row's two sums with two rows an SM.  One row: 2 us, launch to launch.
//
// dw and db are sums down the columns: a thread has the same columns of each of its rows, so that its share of both sums stays in
// registers, and one part for each CTA goes to the workspace, which a second kernel adds up: 8 bytes a column and CTA beside 6 a
// column and row.  The order of the sums depends on the sizes alone.  8192 x 4096 bf16: 41 to 44 us, 4.5 to 4.9 TB/s; 41 of them are the
// first kernel's, at 2.5 instructions a cycle and 51 % of the memory's peak, with three rows an SM.
#include "../clpk_activation.cuh"
#include "../clpk_elements.cuh"
#include "../clpk_internal.h"
#include "../clpk_ptx.cuh"

#include <algorithm>
#include <cmath>

namespace clpk {

// Two sums with one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

struct NormParams {
    const void *x, *weight, *bias;
    void *y;
    float *mean, *rstd;
    uint64_t ldx, ldy;
    uint32_t m, d;
    float eps, one_of_d;                            // 1 / d
    // 1 / d in two parts, for the mean: a quotient to 2^-46, so that the mean of equal elements is one of them wherever their sum is exact.
    // The first is rounded down and the second above 0, for an infinite sum to stay infinite.
    float one_of_d_low, one_of_d_rest;
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

// 1 / sqrt of the variance and eps.  There is none where the squares have gone beyond fp32, and the row is NaN (inf * 0): with the 0 that
// 1 / sqrt(inf) is, it would come out as its bias.
__device__ __forceinline__ float row_rstd(float variance) { return 1.0f / sqrtf(fmaf(variance, 0.0f, variance)); }

// Eight elements of a row, or as many as a vector has: what a thread loads at a time
template <int DT> constexpr int kPiece = Element<DT>::kPerVector;

// weights of a piece in fp32, two by two; `none` where there are none
template <int WDT, int PAIRS>
__device__ __forceinline__ void load_weights(float2 (&w)[PAIRS], const void *base, uint32_t at, uint32_t d, float none)
{
    constexpr int N = 2 * PAIRS;
    if (!base) {
#pragma unroll
        for (int j = 0; j < PAIRS; j++)
            w[j] = make_float2(none, none);
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

// ---- rows ahead ----------------------------------------------------------------------------------------------
//
// A thread's share of a row is asked for some rows ahead, into shared memory that is the thread's own: what it reads there it has copied
// there itself, so that no thread waits for another, and no register holds what is on its way.

__device__ __forceinline__ void ask_piece(void *to, const void *from, uint32_t bytes)       // 16, or fewer and zeros behind them
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void asked()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void wait_asked()                    // all but the last N groups are there
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The pieces of rows that fall to a thread, one row after another: `at`, the thread's first piece of the next row, and how many bytes of each
// piece there are.
template <int DT, int THREADS, int PIECES> struct RowsAhead {
    static constexpr uint32_t N = kPiece<DT>;
    const typename Element<DT>::T *at;
    uint64_t step;                                              // elements to the next row
    uint32_t bytes[PIECES];

    __device__ __forceinline__ RowsAhead(const void *base, uint64_t ld, uint64_t first, uint64_t rows, uint32_t t, uint32_t d)
        : at(static_cast<const typename Element<DT>::T *>(base) + first * ld + t * N), step(rows * ld)
    {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const uint32_t from = (i * THREADS + t) * N;
            bytes[i] = from >= d ? 0 : min(d - from, N) * (16 / N);
        }
    }
    template <uint32_t STRIDE> __device__ __forceinline__ void ask(uint4 *to)
    {
#pragma unroll
        for (int i = 0; i < PIECES; i++)
            if (bytes[i])
                ask_piece(to + i * STRIDE, at + i * THREADS * N, bytes[i]);
        at += step;
    }
};

constexpr int kNormWarps = 4;                       // rows that a CTA takes at once where a row is a warp's
constexpr int kNormAhead = 2;                       // rows on their way behind the one that is computed

// How many CTAs an SM holds: 128 registers a thread for 32 elements with their weights, 80 and 56 for 16 and 8 (with 48, for ten, some are
// spilled: 65536 x 256 bf16 16.3 us, so 15.0).
__host__ __device__ constexpr int norm_ctas(int threads, int elems)
{
    return threads == 32 ? (elems == 32 ? 4 : elems == 16 ? 6 : 9) : (elems == 32 ? 512 : 768) / threads;
}
template <int DT> constexpr uint32_t norm_bytes(int threads, int elems)
{
    return (kNormAhead + 1) * (threads == 32 ? 32 * kNormWarps : threads) * elems * (uint32_t)sizeof(typename Element<DT>::T);
}

// THREADS share a row of up to THREADS * ELEMS elements; rows and weights start on 16 bytes
template <int DT, int WDT, int THREADS, int ELEMS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kNormWarps : THREADS, norm_ctas(THREADS, ELEMS)) layer_norm_kernel(NormParams p)
{
    using T = typename Element<DT>::T;
    constexpr int N = kPiece<DT>, kPieces = ELEMS / N, kRows = THREADS == 32 ? kNormWarps : 1;
    constexpr uint32_t kAll = THREADS == 32 ? 32 * kNormWarps : THREADS, kStage = kPieces * kAll;
    extern __shared__ __align__(16) uint4 ring[];
    __shared__ float shared[2][THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t t = threadIdx.x % THREADS, step = gridDim.x * kRows;
    const uint64_t first = blockIdx.x * kRows + (THREADS == 32 ? threadIdx.x >> 5 : 0);
    uint4 *const mine = ring + threadIdx.x;
    RowsAhead<DT, THREADS, kPieces> ahead(p.x, p.ldx, first, step, t, p.d);
    const auto ask = [&](uint64_t row, uint32_t stage) {
        if (row < p.m)
            ahead.template ask<kAll>(mine + stage * kStage);
        asked();
    };
#pragma unroll
    for (uint32_t i = 0; i < kNormAhead; i++)
        ask(first + (uint64_t)i * step, i);
    float2 w[ELEMS / 2], b[ELEMS / 2];
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const uint32_t at = (i * THREADS + t) * N;
        load_weights<WDT>(reinterpret_cast<float2(&)[N / 2]>(w[i * N / 2]), p.weight, at, p.d, 1.0f);
        load_weights<WDT>(reinterpret_cast<float2(&)[N / 2]>(b[i * N / 2]), p.bias, at, p.d, 0.0f);
    }
    T *y = static_cast<T *>(p.y) + first * p.ldy + t * N;
    uint32_t stage = 0;
    for (uint64_t row = first; row < p.m; row += step) {
        ask(row + (uint64_t)kNormAhead * step, stage == 0 ? kNormAhead : stage - 1);
        wait_asked<kNormAhead>();
        Raw<DT, N> raw[kPieces];
        float2 sum = make_float2(0.0f, 0.0f), squares = sum;
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t at = (i * THREADS + t) * N;
            raw[i].v[0] = at < p.d ? mine[stage * kStage + i * kAll] : make_uint4(0, 0, 0, 0);
            float2 v[N / 2];
            raw[i].widen(v);
#pragma unroll
            for (int j = 0; j < N / 2; j++)
                sum = add2(sum, v[j]);
        }
        const float all = row_sum<THREADS>(sum.x + sum.y, shared[0]), mean = fmaf(all, p.one_of_d_low, all * p.one_of_d_rest);
        const float2 minus = make_float2(-mean, -mean);
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t at = (i * THREADS + t) * N;
            float2 v[N / 2];
            raw[i].widen(v);
            if (at + N <= p.d) {
#pragma unroll
                for (int j = 0; j < N / 2; j++) {
                    const float2 off = add2(v[j], minus);
                    squares = fma2(off, off, squares);
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float off = (j % 2 ? v[j / 2].y : v[j / 2].x) - mean;
                    squares.x = at + j < p.d ? fmaf(off, off, squares.x) : squares.x;
                }
            }
        }
        const float rstd = row_rstd(row_sum<THREADS>(squares.x + squares.y, shared[1]) * p.one_of_d + p.eps);
        if (t == 0) {
            if (p.mean)
                p.mean[row] = mean;
            if (p.rstd)
                p.rstd[row] = rstd;
        }
        const float2 scale = make_float2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            const uint32_t at = (i * THREADS + t) * N;
            if (at >= p.d)
                break;
            float2 v[N / 2];
            raw[i].widen(v);
#pragma unroll
            for (int j = 0; j < N / 2; j++)
                v[j] = fma2(mul2(add2(v[j], minus), scale), w[i * N / 2 + j], b[i * N / 2 + j]);
            raw[i].round(v);
            if (at + N <= p.d)
                raw[i].store(y + i * THREADS * N);
            else
                raw[i].store_some(y + i * THREADS * N, p.d - at);
        }
        y += step * p.ldy;
        stage = stage == kNormAhead ? 0 : stage + 1;
    }
    wait_asked<0>();
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
    const float rstd = row_rstd(row_sum<256>(squares, shared[1]) / (float)p.d + p.eps);
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
    float one_of_d;                                 // 1 / d
};

// Sums of V values each over all threads of a row, which are a CTA or group `group` of it.  Lanes halve what they add: each sends the values
// that the other half of a warp goes on with, so that V values take little more than one.  `shared`: V words for each warp, not to be
// written again before all threads have come to the next barrier.
template <int THREADS, int V>
__device__ __forceinline__ void row_sums(float (&v)[V], float *shared, uint32_t group)
{
    const uint32_t lane = threadIdx.x & 31;
    int o = 16;
#pragma unroll
    for (int left = V / 2; left > 0; left /= 2, o /= 2) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < left; i++) {
            const float keep = upper ? v[left + i] : v[i], give = upper ? v[i] : v[left + i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    constexpr uint32_t kEach = 32 / V;                          // lanes that have the same value now, value i from lane i * kEach on
#pragma unroll
    for (uint32_t x = kEach / 2; x > 0; x /= 2)
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], x);
    if constexpr (THREADS == 32) {
#pragma unroll
        for (int i = V - 1; i >= 0; i--)
            v[i] = __shfl_sync(0xffffffffu, v[0], i * kEach);
    } else {
        constexpr uint32_t kWarps = THREADS / 32;
        if (lane % kEach == 0)
            shared[threadIdx.x % THREADS / 32 * V + lane / kEach] = v[0];
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(THREADS) : "memory");
        float sum = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; w += 32 / V)
            if (w + lane / V < kWarps)
                sum += shared[(w + lane / V) * V + lane % V];
#pragma unroll
        for (uint32_t x = V; x < 32 && x < kWarps * V; x *= 2)
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
#pragma unroll
        for (int i = 0; i < V; i++)
            v[i] = __shfl_sync(0xffffffffu, sum, i);
    }
}

// A CTA for each SM: groups of threads that share a row each, as many as registers (two sums for each element) and shared memory (two rows
// of x and dy at least, and the weights) hold, and rows on their way behind the one that is computed, two at most.
constexpr uint32_t kNormGradBytes = 216 * 1024;
__host__ __device__ constexpr uint32_t norm_grad_row(int threads, int elems, uint32_t elem) { return 2 * threads * elems * elem; }
__host__ __device__ constexpr uint32_t norm_grad_room(int threads, int elems) { return kNormGradBytes - threads * elems * 4; }
__host__ __device__ constexpr int norm_grad_groups(int threads, int elems, uint32_t elem)
{
    int groups = (elems == 8 ? 640 : elems == 32 || threads <= 64 ? 512 : 768) / threads;        // 102, 128 and 85 registers
    while (groups > 1 && groups * 2 * norm_grad_row(threads, elems, elem) > norm_grad_room(threads, elems))
        groups /= 2;
    return groups;
}
__host__ __device__ constexpr int norm_grad_ahead(int threads, int elems, uint32_t elem)
{
    const int rows = norm_grad_room(threads, elems) / (norm_grad_groups(threads, elems, elem) * norm_grad_row(threads, elems, elem));
    return rows >= 3 ? 2 : rows - 1;
}

// The groups' shares of dw and db, one group's behind the other's, to the CTA's part.  Not inlined: beside it the loop over rows gets
// other registers, and mostly takes longer (bf16 8192 x 5120: 60.9 us, so 50.0; 4096 x 8192 49.4 and 40.5; 8192 x 4096 41.1 and 40.7; one row
// of 4096 4.95 and 5.15).
template <uint32_t COLUMNS>
__device__ __noinline__ void add_shares(const float *shares, float *part, uint32_t groups, uint32_t d)
{
    const bool whole = d % 4 == 0;
#pragma unroll 2
    for (uint32_t i = 4 * threadIdx.x; i < 2 * COLUMNS; i += 4 * blockDim.x) {
        const uint32_t at = i % COLUMNS;
        if (at >= d)
            continue;
        float4 sum = *reinterpret_cast<const float4 *>(shares + i);
#pragma unroll 4
        for (uint32_t g = 1; g < groups; g++) {
            const float4 f = *reinterpret_cast<const float4 *>(shares + g * 2 * COLUMNS + i);
            sum = make_float4(sum.x + f.x, sum.y + f.y, sum.z + f.z, sum.w + f.w);
        }
        float *const to = part + i / COLUMNS * d + at;
        if (whole) {
            *reinterpret_cast<float4 *>(to) = sum;
        } else {
            const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (at + j < d)
                    to[j] = v[j];
        }
    }
}

template <int DT, int WDT, int THREADS, int ELEMS>
__global__ void __launch_bounds__(THREADS * norm_grad_groups(THREADS, ELEMS, sizeof(typename Element<DT>::T)), 1) layer_norm_gradients_kernel(NormGradParams p)
{
    using T = typename Element<DT>::T;
    constexpr int N = kPiece<DT>, kPieces = ELEMS / N, kGroups = norm_grad_groups(THREADS, ELEMS, sizeof(T)), kAhead = norm_grad_ahead(THREADS, ELEMS, sizeof(T));
    constexpr uint32_t kAll = THREADS * kGroups, kRow = 2 * kPieces * kAll;     // also where fewer groups run
    extern __shared__ __align__(16) uint4 ring[];
    __shared__ float shared[2][kGroups][THREADS / 32 * 2];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t group = threadIdx.x / THREADS, t = threadIdx.x % THREADS, groups = blockDim.x / THREADS, step = gridDim.x * groups;
    const uint64_t first = blockIdx.x * groups + group;
    uint4 *const mine = ring + threadIdx.x;
    RowsAhead<DT, THREADS, kPieces> ahead_x(p.x, p.ldx, first, step, t, p.d), ahead_dy(p.dy, p.lddy, first, step, t, p.d);
    const auto ask = [&](uint64_t row, uint32_t turn) {
        if (row < p.m) {
            ahead_x.template ask<kAll>(mine + turn * kRow);
            ahead_dy.template ask<kAll>(mine + turn * kRow + kPieces * kAll);
        }
        asked();
    };
    // Behind a row x and dy are zeros, here and as the copies fill them up: what they bring to a sum is zero, but for a row that is NaN in
    // any case.
#pragma unroll
    for (int i = 0; i < kPieces; i++)
        if (ahead_x.bytes[i] == 0)
            for (uint32_t turn = 0; turn <= kAhead; turn++)
                mine[turn * kRow + i * kAll] = mine[turn * kRow + (kPieces + i) * kAll] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (uint32_t i = 0; i < kAhead; i++)
        ask(first + (uint64_t)i * step, i);
    // the weights of a thread's elements, four by four: in shared memory, where they take no registers from the sums (8192 x 4096 bf16: 6 us)
    float4 *const weights = reinterpret_cast<float4 *>(ring + (kAhead + 1) * kRow) + t;
    if (group == 0) {
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            float2 w[N / 2];
            load_weights<WDT>(w, p.weight, (i * THREADS + t) * N, p.d, 1.0f);
#pragma unroll
            for (int j = 0; j < N / 4; j++)
                weights[(i * N / 4 + j) * THREADS] = make_float4(w[2 * j].x, w[2 * j].y, w[2 * j + 1].x, w[2 * j + 1].y);
        }
    }
    __syncthreads();
    float2 dw[ELEMS / 2] = {}, db[ELEMS / 2] = {};
    T *dx = static_cast<T *>(p.dx) + first * p.lddx + t * N;
    uint32_t turn = 0, flip = 0;
    float mean = first < p.m ? p.mean[first] : 0.0f, rstd = first < p.m ? p.rstd[first] : 0.0f;
    for (uint64_t row = first; row < p.m; row += step) {
        ask(row + (uint64_t)kAhead * step, turn == 0 ? kAhead : turn - 1);
        const bool more = row + step < p.m;
        const float next_mean = more ? p.mean[row + step] : 0.0f, next_rstd = more ? p.rstd[row + step] : 0.0f;
        wait_asked<kAhead>();
        // |mean| * rstd beyond fp32 is a row of equal elements, whose xhat is 0: so is what stands for it behind the row's end, -mean * 0
        const float by_hat = fabsf(mean * rstd) > 3.402823466e38f && rstd <= 3.402823466e38f ? 0.0f : rstd;
        const float2 scale = make_float2(by_hat, by_hat);
        // xhat, dy and the weights of a piece, two numbers at a time.  xhat first: dy times x - mean may leave fp32 where dy times xhat does not.
        const auto values = [&](int i, float2 (&hat)[N / 2], float2 (&dy)[N / 2], float2 (&w)[N / 2]) {
            Raw<DT, N> x, d;
            x.v[0] = mine[turn * kRow + i * kAll];
            d.v[0] = mine[turn * kRow + (kPieces + i) * kAll];
#pragma unroll
            for (int j = 0; j < N / 4; j++) {
                const float4 f = weights[(i * N / 4 + j) * THREADS];
                w[2 * j] = make_float2(f.x, f.y);
                w[2 * j + 1] = make_float2(f.z, f.w);
            }
            x.widen(hat);
            d.widen(dy);
#pragma unroll
            for (int j = 0; j < N / 2; j++)
                hat[j] = mul2(add2(hat[j], make_float2(-mean, -mean)), scale);
        };
        float2 sum_g = make_float2(0.0f, 0.0f), sum_gh = sum_g;         // of g and of g * xhat
#pragma unroll
        for (int i = 0; i < kPieces; i++) {
            float2 hat[N / 2], dy[N / 2], w[N / 2];
            values(i, hat, dy, w);
#pragma unroll
            for (int j = 0; j < N / 2; j++) {
                const int e = i * N / 2 + j;
                const float2 both = mul2(dy[j], hat[j]);
                dw[e] = add2(dw[e], both);
                db[e] = add2(db[e], dy[j]);
                sum_g = fma2(dy[j], w[j], sum_g);
                sum_gh = fma2(both, w[j], sum_gh);
            }
        }
        if (p.dx) {
            float sums[2] = {sum_g.x + sum_g.y, sum_gh.x + sum_gh.y};
            row_sums<THREADS, 2>(sums, shared[flip][group], group);
            flip ^= 1;
            // dx = rstd g + xhat by + also, by = -rstd * mean(g xhat), also = -rstd * mean(g)
            const float by = -rstd * (sums[1] * p.one_of_d), also = -rstd * (sums[0] * p.one_of_d);
            asm volatile("" ::: "memory");                      // all is read again rather than kept in registers
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                if (ahead_x.bytes[i] == 0)
                    break;
                float2 hat[N / 2], dy[N / 2], w[N / 2];
                values(i, hat, dy, w);
#pragma unroll
                for (int j = 0; j < N / 2; j++)
                    hat[j] = fma2(mul2(dy[j], w[j]), make_float2(rstd, rstd), fma2(hat[j], make_float2(by, by), make_float2(also, also)));
                Raw<DT, N> out;
                out.round(hat);
                if (ahead_x.bytes[i] == 16)
                    out.store(dx + i * THREADS * N);
                else
                    out.store_some(dx + i * THREADS * N, ahead_x.bytes[i] / (16 / N));
            }
            dx += step * p.lddx;
        }
        mean = next_mean;
        rstd = next_rstd;
        turn = turn == kAhead ? 0 : turn + 1;
    }
    wait_asked<0>();
    if (!p.parts)
        return;
    // the groups' shares side by side where the rows were, each in the order of its columns, then added in their order
    constexpr uint32_t kColumns = THREADS * ELEMS;
    float *const shares = reinterpret_cast<float *>(ring);
    static_assert(sizeof(float) <= (kAhead + 1) * sizeof(T), "room for all shares");
    static_assert(THREADS == 32 || kGroups < 16, "barriers of a CTA");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPieces; i++)
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
            const int e = i * N / 2 + 2 * j;
            float4 *const to = reinterpret_cast<float4 *>(shares + group * 2 * kColumns + (i * THREADS + t) * N) + j;
            to[0] = make_float4(dw[e].x, dw[e].y, dw[e + 1].x, dw[e + 1].y);
            to[kColumns / 4] = make_float4(db[e].x, db[e].y, db[e + 1].x, db[e + 1].y);
        }
    __syncthreads();
    add_shares<kColumns>(shares, p.parts + (uint64_t)blockIdx.x * 2 * p.d, groups, p.d);
}

// Rows that do not start on 16 bytes, or are too long for registers: dx of a row by a CTA, element by element, read twice
template <int DT, int WDT>
__global__ void __launch_bounds__(256) layer_norm_plain_dx_kernel(NormGradParams p)
{
    using E = Element<DT>;
    using W = Element<WDT>;
    __shared__ float shared[16];
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
    float sums[2] = {}, hat, g;
#pragma unroll 4
    for (uint64_t at = threadIdx.x; at < p.d; at += 256) {
        values(at, hat, g);
        sums[0] += g;
        sums[1] = fmaf(g, hat, sums[1]);
    }
    row_sums<256, 2>(sums, shared, 0);
    const float c1 = sums[0] * p.one_of_d, c2 = sums[1] * p.one_of_d;
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

// The parts' sums, rounded: a lane has a column, and each of 32 warps every 32nd part, so that all loads are on their way at once
constexpr int kNormJoinWarps = 32;
constexpr uint32_t kNormParts = 148;                // at most
template <int WDT>
__global__ void __launch_bounds__(32 * kNormJoinWarps) layer_norm_join_kernel(NormJoinParams p)
{
    __shared__ float sums[kNormJoinWarps][32];
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane, which = blockIdx.y;
    if (!p.out[which])
        return;
    float sum = 0.0f;
    if (col < p.d) {
        const float *from = p.parts + (uint64_t)which * p.d + col;
        constexpr uint32_t kEach = (kNormParts + kNormJoinWarps - 1) / kNormJoinWarps;
        float part[kEach];
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++)
            part[j] = warp + j * kNormJoinWarps < p.n_parts ? from[(uint64_t)(warp + j * kNormJoinWarps) * 2 * p.d] : 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++)
            sum += part[j];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp > 0 || col >= p.d)
        return;
#pragma unroll
    for (uint32_t w = 1; w < kNormJoinWarps; w++)
        sum += sums[w][lane];
    static_cast<typename Element<WDT>::T *>(p.out[which])[col] = Element<WDT>::round(sum);
}

// ---- host side ------------------------------------------------------------------------------------------

constexpr uint32_t kNormLongest = 16384, kNormGradLongest = 16384;      // elements of a row in registers

template <int DT, int WDT, int THREADS, int ELEMS>
static int launch_norm_rows(const NormParams &p, cudaStream_t s)
{
    constexpr int kThreads = THREADS == 32 ? 32 * kNormWarps : THREADS;
    constexpr uint32_t kBytes = norm_bytes<DT>(THREADS, ELEMS);
    if (kBytes > 47 * 1024)
        CLPK_CUDA(cudaFuncSetAttribute(layer_norm_kernel<DT, WDT, THREADS, ELEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBytes));
    const uint32_t ctas = std::min<uint32_t>(THREADS == 32 ? (p.m - 1) / kNormWarps + 1 : p.m, norm_ctas(THREADS, ELEMS) * (uint32_t)num_sms());
    return launch_behind(layer_norm_kernel<DT, WDT, THREADS, ELEMS>, "layer_norm", ctas, kThreads, kBytes, s, p);
}

// Threads that share a row, and elements of each: what leaves few threads without a part of the row, 16 elements rather than 32 while two
// rows at least fit an SM.  bf16, against 128 and 256 threads of 32 for all: 8192 rows of 2048 12.8 and 20.3 us, of 2560 18.2 and 21.2, of 4096
// 25.0 and 25.1, of 5120 35.5 and 40.4, of 6144 37.9 and 42.0.  Where the SMs take all rows at once a row is for more threads: one of 1024 1.9
// and 2.7 us, but 16384 of 768 12.5 and 11.0.
template <int DT, int WDT>
static int launch_norm(const NormParams &p, bool aligned, cudaStream_t s)
{
    const auto few = [&](int threads, int elems) { return p.m <= norm_ctas(threads, elems) * (uint32_t)num_sms(); };
    if (!aligned || p.d > kNormLongest)
        return launch_behind(layer_norm_plain_kernel<DT, WDT>, "layer_norm_plain", p.m, 256, 0, s, p);
    if (p.d <= 256)
        return launch_norm_rows<DT, WDT, 32, 8>(p, s);
    if (p.d <= 512)
        return launch_norm_rows<DT, WDT, 32, 16>(p, s);
    if (p.d <= 1024)
        return few(64, 16) ? launch_norm_rows<DT, WDT, 64, 16>(p, s) : launch_norm_rows<DT, WDT, 32, 32>(p, s);
    if (p.d <= 2048)
        return launch_norm_rows<DT, WDT, 128, 16>(p, s);
    if (p.d <= 2560)
        return launch_norm_rows<DT, WDT, 160, 16>(p, s);
    if (p.d <= 4096)
        return launch_norm_rows<DT, WDT, 256, 16>(p, s);
    if (p.d <= 5120)
        return launch_norm_rows<DT, WDT, 320, 16>(p, s);
    if (p.d <= 6144)
        return launch_norm_rows<DT, WDT, 384, 16>(p, s);
    if (p.d <= 8192)
        return few(512, 16) ? launch_norm_rows<DT, WDT, 512, 16>(p, s) : launch_norm_rows<DT, WDT, 256, 32>(p, s);
    return launch_norm_rows<DT, WDT, 512, 32>(p, s);
}

// Threads and elements of each that share a row in layer_norm_gradients_kernel: as above.  bf16, 8192 rows: of 2560 27.8 us, with 256 threads
// 35.9; of 5120 50.0, with 384 54.4; of 5128 57.2, with 256 of 32 elements 59.2, of 6144 58.6 and 57.9 (fp32 93.3 and 93.2, 110 and 100; 20 rows
// of 6144 7.8 and 8.1).
struct NormGradShape {
    int threads, elems;
};
constexpr NormGradShape norm_grad_shape(uint32_t d)
{
    return d <= 256 ? NormGradShape{32, 8} : d <= 512 ? NormGradShape{32, 16} : d <= 1024 ? NormGradShape{64, 16} : d <= 2048 ? NormGradShape{128, 16}
         : d <= 2560 ? NormGradShape{160, 16} : d <= 4096 ? NormGradShape{256, 16} : d <= 5120 ? NormGradShape{320, 16} : d <= 6144 ? NormGradShape{384, 16}
         : d <= 8192 ? NormGradShape{256, 32} : NormGradShape{512, 32};
}

// Groups of a CTA, and the CTAs that share the rows, each with a part of dw and db.  Few rows are spread over the SMs.  A whole B200's SMs:
// the workspace's size may not depend on the card at hand.
static uint32_t norm_groups(uint32_t m, uint32_t d, uint64_t elem)
{
    const NormGradShape shape = norm_grad_shape(d);
    return std::min((uint32_t)norm_grad_groups(shape.threads, shape.elems, (uint32_t)elem), m ? (m - 1) / kNormParts + 1 : 1);
}
static uint32_t norm_parts(uint32_t m, uint32_t d, uint64_t elem)
{
    return std::min(m ? (m - 1) / norm_groups(m, d, elem) + 1 : 1, kNormParts);
}

template <int DT, int WDT, int THREADS, int ELEMS>
static int launch_norm_gradient_rows(const NormGradParams &p, uint32_t parts, cudaStream_t s)
{
    constexpr uint32_t kElem = sizeof(typename Element<DT>::T), kEach = (norm_grad_ahead(THREADS, ELEMS, kElem) + 1) * norm_grad_row(THREADS, ELEMS, kElem);
    constexpr uint32_t kMost = norm_grad_groups(THREADS, ELEMS, kElem) * kEach + THREADS * ELEMS * 4;
    if (kMost > 40 * 1024)
        CLPK_CUDA(cudaFuncSetAttribute(layer_norm_gradients_kernel<DT, WDT, THREADS, ELEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost));
    const uint32_t groups = norm_groups(p.m, p.d, kElem);
    return launch_behind(layer_norm_gradients_kernel<DT, WDT, THREADS, ELEMS>, "layer_norm_gradients", parts, groups * THREADS, kMost, s, p);
}

template <int DT, int WDT>
static int launch_norm_gradients(const NormGradParams &p, bool aligned, uint32_t parts, cudaStream_t s)
{
    if (!aligned || p.d > kNormGradLongest) {
        if (p.dx)
            CLPK_TRY(launch_behind(layer_norm_plain_dx_kernel<DT, WDT>, "layer_norm_plain_dx", p.m, 256, 0, s, p));
        return p.parts ? launch_behind(layer_norm_plain_columns_kernel<DT>, "layer_norm_plain_columns", dim3((p.d - 1) / 256 + 1, parts), 256, 0, s, p) : CLPK_OK;
    }
    const NormGradShape shape = norm_grad_shape(p.d);
    if (shape.elems == 8)
        return launch_norm_gradient_rows<DT, WDT, 32, 8>(p, parts, s);
    if (shape.elems == 32)
        return shape.threads == 256 ? launch_norm_gradient_rows<DT, WDT, 256, 32>(p, parts, s) : launch_norm_gradient_rows<DT, WDT, 512, 32>(p, parts, s);
    switch (shape.threads) {
    case 32:  return launch_norm_gradient_rows<DT, WDT, 32, 16>(p, parts, s);
    case 64:  return launch_norm_gradient_rows<DT, WDT, 64, 16>(p, parts, s);
    case 128: return launch_norm_gradient_rows<DT, WDT, 128, 16>(p, parts, s);
    case 160: return launch_norm_gradient_rows<DT, WDT, 160, 16>(p, parts, s);
    case 256: return launch_norm_gradient_rows<DT, WDT, 256, 16>(p, parts, s);
    case 320: return launch_norm_gradient_rows<DT, WDT, 320, 16>(p, parts, s);
    default:  return launch_norm_gradient_rows<DT, WDT, 384, 16>(p, parts, s);
    }
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
    return (uint64_t)std::min(std::max(m, 1u), kNormParts) * 2 * d * sizeof(float);
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
    const float near = (float)(1.0 / a.d), low = (double)near > 1.0 / a.d ? std::nextafterf(near, 0.0f) : near;
    const NormParams p = {a.d_x, a.d_weight, a.d_bias, a.d_y, a.d_mean, a.d_rstd, a.ldx, a.ldy, a.m, a.d, a.eps, near, low, std::max((float)(1.0 / a.d - low), 1e-37f)};
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
    const uint32_t parts = norm_parts(a.m, a.d, element_bytes(a.dtype));
    const uint64_t need = norm_workspace(a.m, a.d);
    CLPK_REQUIRE(!columns || (a.d_workspace && a.workspace_bytes >= need && (uintptr_t)a.d_workspace % 16 == 0), "%s: needs a 16-byte aligned workspace of %llu bytes",
                 what, (unsigned long long)need);
    const NormGradParams p = {a.d_x, a.d_weight, a.d_dy, a.d_mean, a.d_rstd, a.d_dx, columns ? static_cast<float *>(a.d_workspace) : nullptr,
                              a.ldx, a.lddy, a.lddx, a.m, a.d, (float)(1.0 / a.d)};
    const int rc = CLPK_BY_TYPES(a.dtype, a.weight_dtype, launch_norm_gradients, p, aligned, parts, s);
    if (rc != CLPK_OK || !columns)
        return rc;
    const NormJoinParams join = {p.parts, {a.d_dweight, a.d_dbias}, parts, a.d};
    const dim3 grid((a.d - 1) / 32 + 1, 2);
    constexpr int kThreads = 32 * kNormJoinWarps;
    switch (a.weight_dtype) {
    case CLPK_DT_F32: return launch_behind(layer_norm_join_kernel<CLPK_DT_F32>, "layer_norm_join", grid, kThreads, 0, s, join);
    case CLPK_DT_F16: return launch_behind(layer_norm_join_kernel<CLPK_DT_F16>, "layer_norm_join", grid, kThreads, 0, s, join);
    default:          return launch_behind(layer_norm_join_kernel<CLPK_DT_BF16>, "layer_norm_join", grid, kThreads, 0, s, join);
    }
}

} // extern "C"
