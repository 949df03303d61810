// Activations of a gated feed-forward layer and their derivatives, in fp32.
//
// exp(x) is ex2.approx of x * log2(e): the rounding of that product costs a relative error that grows with |x| to 5e-6 at |x| = 88,
// where the sigmoid it stands in has long been 0 or 1; below |x| = 8 it is under 5e-7.  Quotients are products with rcp.approx (1
// ulp).  Both flush what is below 2^-126 to 0, which 1 + exp(x) does not see and 1 / (1 + exp(x)) is not missed in; without
// that each takes three instructions more.  tanh-GELU is a sigmoid too: (1 + tanh y) / 2 = 1 / (1 + exp(-2 y)).
// An element then takes two special-function results, sixteen cycles of a scheduler, and three other instructions (activate2).
//
// GELU's normal distribution function is Abramowitz and Stegun 7.1.26: erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + p x),
// x >= 0, off by 1.5e-7 at most; in fp32 the function is within 3.0e-7 and GELU within 4.2e-7, which is what erff and its sum with 1
// lose too (4.5e-7).  Below 0, where that sum cancels, the error here falls with exp(-x^2) (g = -5: -1.4355e-6 for -1.4332e-6,
// with erff -1.4901e-6).  In place of erff it took gated bf16 4096 x 512 x 4096 from 38.2 to 35.0 us and int8 1378 x 144 x 13968 from 45.4
// to 39.0, with eight epilogue warps; with sixteen they take 29 and 29, and 28.5 and 22 with ReLU.
#pragma once

#include <stdint.h>

#include "../../include/clpeak_b200_kernels.h"

namespace clpk {

constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float exp_approx(float x) { return ex2_approx(x * kLog2E); }

__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float sigmoid(float x) { return rcp_approx(1.0f + exp_approx(-x)); }

// a NaN stays one
__device__ __forceinline__ float relu(float g)
{
    float y;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(g));
    return y;
}

// g in [-most, most]; a NaN stays one
__device__ __forceinline__ float clamped(float g, float most)
{
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(g), "f"(most));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(y), "f"(-most));
    return y;
}

constexpr float kGeluC = 0.7978845608028654f;       // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

constexpr float kSqrtHalf = 0.7071067811865476f;
constexpr float kErfP = 0.3275911f, kErf1 = 0.254829592f, kErf2 = -0.284496736f, kErf3 = 1.421413741f, kErf4 = -1.453152027f, kErf5 = 1.061405429f;

// (1 + erf(g / sqrt(2))) / 2, and exp(-g^2 / 2)
__device__ __forceinline__ float normal_cdf(float g, float &e)
{
    const float x = fabsf(g) * kSqrtHalf, t = rcp_approx(1.0f + kErfP * x);
    e = exp_approx(-0.5f * g * g);
    const float q = 0.5f * e * t * (kErf1 + t * (kErf2 + t * (kErf3 + t * (kErf4 + t * kErf5))));
    return g < 0.0f ? q : 1.0f - q;
}

template <int ACT>
__device__ __forceinline__ float activate(float g)
{
    if constexpr (ACT == CLPK_ACT_SILU)
        return g * sigmoid(g);
    else if constexpr (ACT == CLPK_ACT_GELU_TANH)
        return g * sigmoid(2.0f * kGeluC * g * (1.0f + kGeluCubic * g * g));
    else if constexpr (ACT == CLPK_ACT_GELU) {
        float e;
        return g * normal_cdf(g, e);
    }
    else if constexpr (ACT == CLPK_ACT_RELU)
        return relu(g);
    else
        return sigmoid(g);
}

// Two floats with one instruction.  act(g) of two: sums and products of two take half the issue slots, which the special-function
// results leave too few of (gated bf16 4096 x 128 x 14336 with GELU 67 -> 63 us, with its tanh form 60 -> 55).
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 c;
    asm("{\n\t"
        ".reg .b64 a, b;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t"
        "}\n"
        : "=f"(c.x), "=f"(c.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    asm("{\n\t"
        ".reg .b64 a, b, c;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, a, b, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t"
        "}\n"
        : "+f"(c.x), "+f"(c.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// 1 / (1 + 2^y)
__device__ __forceinline__ float2 sigmoid2_of(float2 y)
{
    const float2 d = fma2(make_float2(ex2_approx(y.x), ex2_approx(y.y)), both(1.0f), both(1.0f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}

template <int ACT>
__device__ __forceinline__ float2 activate2(float2 g)
{
    if constexpr (ACT == CLPK_ACT_SILU) {
        return mul2(g, sigmoid2_of(mul2(g, both(-kLog2E))));
    } else if constexpr (ACT == CLPK_ACT_GELU_TANH) {
        const float2 cubic = fma2(mul2(g, g), both(kGeluCubic), both(1.0f));
        return mul2(g, sigmoid2_of(mul2(mul2(g, both(-2.0f * kGeluC * kLog2E)), cubic)));
    } else if constexpr (ACT == CLPK_ACT_GELU) {
        const float2 d = fma2(make_float2(fabsf(g.x), fabsf(g.y)), both(kErfP * kSqrtHalf), both(1.0f));
        const float2 t = make_float2(rcp_approx(d.x), rcp_approx(d.y)), y = mul2(mul2(g, both(-0.5f * kLog2E)), g);
        float2 q = fma2(t, both(kErf5), both(kErf4));
        q = fma2(t, q, both(kErf3));
        q = fma2(t, q, both(kErf2));
        q = fma2(t, q, both(kErf1));
        q = mul2(mul2(q, t), mul2(make_float2(ex2_approx(y.x), ex2_approx(y.y)), both(0.5f)));
        return mul2(g, make_float2(g.x < 0.0f ? q.x : 1.0f - q.x, g.y < 0.0f ? q.y : 1.0f - q.y));
    } else if constexpr (ACT == CLPK_ACT_RELU) {
        return make_float2(relu(g.x), relu(g.y));
    } else {
        return sigmoid2_of(mul2(g, both(-kLog2E)));
    }
}

// act(g) and act'(g).  Both are NaN where g is one: dWg says so too then, and not only dx and dWu.
template <int ACT>
__device__ __forceinline__ void activate_both(float g, float &a, float &da)
{
    if constexpr (ACT == CLPK_ACT_SILU) {
        const float p = sigmoid(g);
        a = g * p;
        da = p * (1.0f + g * (1.0f - p));
    } else if constexpr (ACT == CLPK_ACT_GELU_TANH) {
        const float c = clamped(g, 30.0f);                          // beyond, p is 0 or 1 and the second term 0, whatever its factors
        const float p = sigmoid(2.0f * kGeluC * c * (1.0f + kGeluCubic * c * c));
        a = g * p;
        da = p + c * p * (1.0f - p) * (2.0f * kGeluC) * (1.0f + 3.0f * kGeluCubic * c * c);
    } else if constexpr (ACT == CLPK_ACT_GELU) {
        float e;
        const float cdf = normal_cdf(g, e);
        a = g * cdf;
        da = cdf + g * e * 0.3989422804014327f;                     // 1 / sqrt(2 pi)
    } else if constexpr (ACT == CLPK_ACT_RELU) {
        a = relu(g);
        da = g > 0.0f ? 1.0f : a;                                   // a: 0 or NaN
    } else {
        const float p = sigmoid(g);
        a = p;
        da = p * (1.0f - p);
    }
}

} // namespace clpk
