// One scale for each row and 8-bit integers: what stands in front of an 8-bit product with scales for each token and channel.
//
//   scale = max |x| / 127,   q = rint(x * (1 / scale))
//
// Every element is read once: a row stays in the registers of the 32 or 256 threads that share it, as the vectors it was
// loaded in, while they find its largest element.  That is a maximum over the bits of |x|, which order like the values and put
// infinities and NaNs above them, so that one comparison tells a row that has any.  A rounded quotient is the low byte of
// x * r + 1.5 * 2^23: one multiplication, one addition and three quarters of a byte permutation per element.
//
// Bound by memory, e + 1 bytes per element: fp32 4097 x 11007 in 38.2 us (5.9 TB/s), fp16 16384 x 16384 in 118 us (6.8), one token of
// 4096 in 2.5 us, which is the launch.  256 threads with up to sixteen vectors each rather than 1024 with four: a row of
// 1024 was alone on its SM, which then loaded, and then wrote (60.5 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../clpk_internal.h"
#include "../clpk_ptx.cuh"

namespace clpk {

template <int DT> struct RowElem;
template <> struct RowElem<CLPK_DT_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(uint32_t w, int) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t abs_max(uint32_t top, uint32_t w) { return max(top, w & 0x7FFFFFFFu); }
    static __device__ __forceinline__ uint32_t fold(uint32_t top) { return top; }
};
// the 16-bit types: two elements a word; `fold` widens the larger one to the bits of an fp32 number
template <int DT> struct RowElem16 {
    static __device__ __forceinline__ uint32_t abs_max(uint32_t top, uint32_t w) { return __vmaxu2(top, w & 0x7FFF7FFFu); }
    static __device__ __forceinline__ float get(uint32_t w, int j)
    {
        const uint16_t h = (uint16_t)(w >> (16 * j));
        if constexpr (DT == CLPK_DT_BF16)
            return __uint_as_float((uint32_t)h << 16);
        else
            return __half2float(__ushort_as_half(h));
    }
    static __device__ __forceinline__ uint32_t fold(uint32_t top) { return __float_as_uint(get(max(top & 0xFFFFu, top >> 16), 0)); }
};
template <> struct RowElem<CLPK_DT_BF16> : RowElem16<CLPK_DT_BF16> {
    typedef uint16_t T;
};
template <> struct RowElem<CLPK_DT_F16> : RowElem16<CLPK_DT_F16> {
    typedef uint16_t T;
};

struct RowParams {
    int8_t *q;
    float *scales;
    const void *src;
    uint64_t rows, cols, ld_q, ld_src;
};

constexpr float kRoundToByte = 12582912.0f;             // 1.5 * 2^23: the sum's last place is 1

// 1 / scale, or 0 for a row that has none; `top`: the bits of the row's largest |x|
__device__ __forceinline__ float row_scale(uint32_t top, float &scale)
{
    if (top >= 0x7F800000u) {                           // an infinity or a NaN
        scale = __uint_as_float(0x7FC00000u);
        return 0.0f;
    }
    scale = __fdiv_rn(__uint_as_float(top), 127.0f);
    if (scale < 1.17549435e-38f) {
        scale = 0.0f;
        return 0.0f;
    }
    return __frcp_rn(scale);
}

__device__ __forceinline__ uint32_t quotient(float x, float r) { return __float_as_uint(__fadd_rn(__fmul_rn(x, r), kRoundToByte)); }

// the largest of all threads of a row; `shared`: a word per warp
template <int THREADS>
__device__ __forceinline__ uint32_t row_max(uint32_t top, uint32_t *shared)
{
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (THREADS > 32) {
        const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0)
            shared[warp] = top;
        __syncthreads();
        top = __reduce_max_sync(0xffffffffu, lane < THREADS / 32 ? shared[lane] : 0u);
    }
    return top;
}

// THREADS share a row of at most THREADS * VECTORS vectors of 16 bytes; a block of 32-thread rows has four of them
template <int DT, int THREADS, int VECTORS>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) quantize_rows_kernel(RowParams p)
{
    using E = RowElem<DT>;
    constexpr int kPerVector = 16 / sizeof(typename E::T), kPerWord = kPerVector / 4;
    __shared__ uint32_t shared[THREADS / 32];
    griddep_wait();
    griddep_launch_dependents();
    const uint64_t row = THREADS == 32 ? (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    const uint32_t t = threadIdx.x % THREADS;
    if (row >= p.rows)                                  // whole warps, and THREADS == 32 alone: no barrier follows
        return;
    const typename E::T *src = static_cast<const typename E::T *>(p.src) + row * p.ld_src;
    int8_t *q = p.q + row * p.ld_q;

    uint32_t w[VECTORS][4], top = 0;
#pragma unroll
    for (int i = 0; i < VECTORS; i++) {
        const uint64_t at = ((uint64_t)i * THREADS + t) * kPerVector;
        w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0;
        if (at + kPerVector <= p.cols) {
            const uint4 v = *reinterpret_cast<const uint4 *>(src + at);
            w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
        } else if (at < p.cols) {
#pragma unroll
            for (int j = 0; j < kPerVector; j++)
                if (at + j < p.cols) {
                    if constexpr (kPerWord == 1)
                        w[i][j] = __float_as_uint(src[at + j]);
                    else
                        w[i][j / 2] |= (uint32_t)src[at + j] << (16 * (j & 1));
                }
        }
    }
#pragma unroll
    for (int i = 0; i < VECTORS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            top = E::abs_max(top, w[i][j]);
    top = row_max<THREADS>(E::fold(top), shared);
    float scale;
    const float r = row_scale(top, scale);
    if (t == 0)
        p.scales[row] = scale;
    const bool none = top >= 0x7F800000u;
#pragma unroll
    for (int i = 0; i < VECTORS; i++) {
        const uint64_t at = ((uint64_t)i * THREADS + t) * kPerVector;
        uint32_t out[kPerWord];
#pragma unroll
        for (int o = 0; o < kPerWord; o++) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                b[j] = quotient(E::get(w[i][o * (4 / kPerWord) + j / kPerWord], j % kPerWord), r);
            out[o] = none ? 0u : __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
        if (at + kPerVector <= p.cols) {
            if constexpr (kPerWord == 1)
                *reinterpret_cast<uint32_t *>(q + at) = out[0];
            else
                *reinterpret_cast<uint2 *>(q + at) = make_uint2(out[0], out[1]);
        } else if (at < p.cols) {
#pragma unroll
            for (int j = 0; j < kPerVector; j++)
                if (at + j < p.cols)
                    q[at + j] = (int8_t)(out[j / 4] >> (8 * (j % 4)));
        }
    }
}

// Rows that are not aligned, or longer than the registers hold: element by element, read twice.  fp32 4096 x 11008 65 us (aligned
// 36), 4096 x 28672 265 us where its bytes take 90.
template <int DT>
__global__ void __launch_bounds__(256) quantize_rows_plain_kernel(RowParams p)
{
    using E = RowElem<DT>;
    __shared__ uint32_t shared[8];
    griddep_wait();
    griddep_launch_dependents();
    const uint64_t row = blockIdx.x;
    const typename E::T *src = static_cast<const typename E::T *>(p.src) + row * p.ld_src;
    int8_t *q = p.q + row * p.ld_q;
    auto word = [&](uint64_t at) {
        if constexpr (sizeof(typename E::T) == 4)
            return __float_as_uint(src[at]);
        else
            return (uint32_t)src[at];
    };
    uint32_t top = 0;
#pragma unroll 8
    for (uint64_t at = threadIdx.x; at < p.cols; at += 256)
        top = E::abs_max(top, word(at));
    top = row_max<256>(E::fold(top), shared);
    float scale;
    const float r = row_scale(top, scale);
    if (threadIdx.x == 0)
        p.scales[row] = scale;
    const bool none = top >= 0x7F800000u;
#pragma unroll 8
    for (uint64_t at = threadIdx.x; at < p.cols; at += 256)
        q[at] = none ? (int8_t)0 : (int8_t)quotient(E::get(word(at), 0), r);
}

constexpr uint64_t kMostVectors = 16;                // that a thread holds

template <int DT, int THREADS>
static int launch_rows(const RowParams &p, uint64_t vectors, cudaStream_t s)
{
    const unsigned grid = (unsigned)(THREADS == 32 ? (p.rows + 3) / 4 : p.rows);
    const int threads = THREADS == 32 ? 128 : THREADS;
    const uint64_t each = (vectors + THREADS - 1) / THREADS;
    if (each <= 1)
        return launch_behind(quantize_rows_kernel<DT, THREADS, 1>, "quantize_rows", grid, threads, 0, s, p);
    if (each <= 2)
        return launch_behind(quantize_rows_kernel<DT, THREADS, 2>, "quantize_rows", grid, threads, 0, s, p);
    if constexpr (THREADS == 32) {                      // four at most, see quantize_rows
        return launch_behind(quantize_rows_kernel<DT, THREADS, 4>, "quantize_rows", grid, threads, 0, s, p);
    } else {
        if (each <= 4)
            return launch_behind(quantize_rows_kernel<DT, THREADS, 4>, "quantize_rows", grid, threads, 0, s, p);
        if (each <= 8)
            return launch_behind(quantize_rows_kernel<DT, THREADS, 8>, "quantize_rows", grid, threads, 0, s, p);
        if (each <= 12)
            return launch_behind(quantize_rows_kernel<DT, THREADS, 12>, "quantize_rows", grid, threads, 0, s, p);
        return launch_behind(quantize_rows_kernel<DT, THREADS, 16>, "quantize_rows", grid, threads, 0, s, p);
    }
}

template <int DT>
static int quantize_rows(const RowParams &p, cudaStream_t s)
{
    constexpr uint64_t elem = sizeof(typename RowElem<DT>::T), per_vector = 16 / elem;
    const uint64_t vectors = (p.cols + per_vector - 1) / per_vector;
    const bool aligned = (uintptr_t)p.src % 16 == 0 && p.ld_src % per_vector == 0 && (uintptr_t)p.q % per_vector == 0 && p.ld_q % per_vector == 0;
    if (!aligned || vectors > kMostVectors * 256)
        return launch_behind(quantize_rows_plain_kernel<DT>, "quantize_rows_plain", (unsigned)p.rows, 256, 0, s, p);
    return vectors <= 4 * 32 ? launch_rows<DT, 32>(p, vectors, s) : launch_rows<DT, 256>(p, vectors, s);
}

} // namespace clpk

using namespace clpk;

extern "C" int clpk_quantize_rows_i8(int8_t *d_q, float *d_scales, const void *d_src, uint64_t rows, uint64_t cols, uint64_t ld_q, uint64_t ld_src,
                                     int dtype, void *stream)
{
    const int rc = require_sm100();
    if (rc != CLPK_OK)
        return rc;
    CLPK_REQUIRE(dtype == CLPK_DT_F32 || dtype == CLPK_DT_F16 || dtype == CLPK_DT_BF16, "clpk_quantize_rows_i8: dtype %d is not F32, F16 or BF16", dtype);
    CLPK_REQUIRE((ld_q == 0 || ld_q >= cols) && (ld_src == 0 || ld_src >= cols), "clpk_quantize_rows_i8: a pitch is shorter than a row of %llu",
                 (unsigned long long)cols);
    CLPK_REQUIRE(rows <= 0x7FFFFFFFull && cols <= 1ull << 40, "clpk_quantize_rows_i8: %llu x %llu is too large", (unsigned long long)rows, (unsigned long long)cols);
    if (rows == 0)
        return CLPK_OK;
    CLPK_REQUIRE(d_scales && (cols == 0 || (d_q && d_src)), "NULL buffer");
    const uint64_t elem = dtype == CLPK_DT_F32 ? 4 : 2;
    CLPK_REQUIRE((uintptr_t)d_src % elem == 0 && (uintptr_t)d_scales % 4 == 0, "clpk_quantize_rows_i8: a buffer is not aligned to its elements");
    const RowParams p = {d_q, d_scales, d_src, rows, cols, ld_q ? ld_q : cols, ld_src ? ld_src : cols};
    switch (dtype) {
    case CLPK_DT_F32: return quantize_rows<CLPK_DT_F32>(p, as_stream(stream));
    case CLPK_DT_F16: return quantize_rows<CLPK_DT_F16>(p, as_stream(stream));
    default:          return quantize_rows<CLPK_DT_BF16>(p, as_stream(stream));
    }
}
