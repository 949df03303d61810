// Elements of 32 and 16 bits in registers: vectors of 16 bytes, and the fp32 numbers that they stand for (layer_norm.cu, adamw.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "clpk_internal.h"

namespace clpk {

template <int DT> struct Element {                              // CLPK_DT_BF16, CLPK_DT_F16
    typedef uint16_t T;
    static constexpr int kPerVector = 8;
    static __device__ __forceinline__ float widen(T x)
    {
        if constexpr (DT == CLPK_DT_BF16)
            return __uint_as_float((uint32_t)x << 16);
        else
            return __half2float(__ushort_as_half(x));
    }
    static __device__ __forceinline__ T round(float x)
    {
        if constexpr (DT == CLPK_DT_BF16)
            return __bfloat16_as_ushort(__float2bfloat16_rn(x));
        else
            return __half_as_ushort(__float2half_rn(x));
    }
    static __device__ __forceinline__ float2 widen2(uint32_t w)
    {
        if constexpr (DT == CLPK_DT_BF16)
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
        else
            return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
    static __device__ __forceinline__ uint32_t round2(float a, float b)
    {
        if constexpr (DT == CLPK_DT_BF16) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
            return *reinterpret_cast<const uint32_t *>(&v);
        } else {
            const __half2 v = __floats2half2_rn(a, b);
            return *reinterpret_cast<const uint32_t *>(&v);
        }
    }
};
template <> struct Element<CLPK_DT_F32> {
    typedef float T;
    static constexpr int kPerVector = 4;
    static __device__ __forceinline__ float widen(T x) { return x; }
    static __device__ __forceinline__ T round(float x) { return x; }
};

// N elements as they lie in memory, in whole vectors
template <int DT, int N> struct Raw {
    static constexpr int kVectors = N / Element<DT>::kPerVector;
    uint4 v[kVectors];

    __device__ __forceinline__ void load(const typename Element<DT>::T *p)
    {
#pragma unroll
        for (int i = 0; i < kVectors; i++)
            v[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    // the first `count` of them, element by element; zeros behind
    __device__ __forceinline__ void load_some(const typename Element<DT>::T *p, uint64_t count)
    {
        uint32_t w[4 * kVectors] = {};
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < count) {
                if constexpr (DT == CLPK_DT_F32)
                    w[j] = __float_as_uint(p[j]);
                else
                    w[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
            }
#pragma unroll
        for (int i = 0; i < kVectors; i++)
            v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    __device__ __forceinline__ void store(typename Element<DT>::T *p) const
    {
#pragma unroll
        for (int i = 0; i < kVectors; i++)
            reinterpret_cast<uint4 *>(p)[i] = v[i];
    }
    __device__ __forceinline__ void store_some(typename Element<DT>::T *p, uint64_t count) const
    {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < count) {
                if constexpr (DT == CLPK_DT_F32)
                    p[j] = __uint_as_float(word(j));
                else
                    p[j] = (uint16_t)(word(j / 2) >> (16 * (j & 1)));
            }
    }
    __device__ __forceinline__ uint32_t word(int i) const
    {
        const uint4 &q = v[i / 4];
        return i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w;
    }
    __device__ __forceinline__ void widen(float (&f)[N]) const
    {
        if constexpr (DT == CLPK_DT_F32) {
#pragma unroll
            for (int j = 0; j < N; j++)
                f[j] = __uint_as_float(word(j));
        } else {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const float2 t = Element<DT>::widen2(word(j / 2));
                f[j] = t.x;
                f[j + 1] = t.y;
            }
        }
    }
    // two by two
    __device__ __forceinline__ void widen(float2 (&f)[N / 2]) const
    {
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            if constexpr (DT == CLPK_DT_F32)
                f[j] = make_float2(__uint_as_float(word(2 * j)), __uint_as_float(word(2 * j + 1)));
            else
                f[j] = Element<DT>::widen2(word(j));
        }
    }
    __device__ __forceinline__ void round(const float2 (&f)[N / 2])
    {
        float one[N];
#pragma unroll
        for (int j = 0; j < N; j++)
            one[j] = j % 2 ? f[j / 2].y : f[j / 2].x;
        round(one);
    }
    __device__ __forceinline__ void round(const float (&f)[N])
    {
        if constexpr (DT == CLPK_DT_F32) {
#pragma unroll
            for (int i = 0; i < kVectors; i++)
                v[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
        } else {
            using E = Element<DT>;
#pragma unroll
            for (int i = 0; i < kVectors; i++)
                v[i] = make_uint4(E::round2(f[8 * i], f[8 * i + 1]), E::round2(f[8 * i + 2], f[8 * i + 3]), E::round2(f[8 * i + 4], f[8 * i + 5]),
                                  E::round2(f[8 * i + 6], f[8 * i + 7]));
        }
    }
};

inline uint64_t element_bytes(int dtype) { return dtype == CLPK_DT_F32 ? 4 : dtype == CLPK_DT_I8 ? 1 : 2; }

} // namespace clpk
