// Activations of a gated feed-forward layer and their derivatives, in fp32.
//
// exp(x) is ex2.approx of x * log2(e): the rounding of that product costs a relative error that grows with |x| to 5e-6 at |x| = 88,
// where the sigmoid it stands in has long been 0 or 1; below |x| = 8 it is under 5e-7.  Quotients are products with rcp.approx (1
// ulp).  Both flush what is below 2^-126 to 0, which 1 + exp(x) does not see and 1 / (1 + exp(x)) is not missed in; without
// that each takes three instructions more.  tanh-GELU is a sigmoid too: (1 + tanh y) / 2 = 1 / (1 + exp(-2 y)).
// An element then takes two special-function results, sixteen cycles of a scheduler, and six other instructions.
//
// GELU's normal distribution function is Abramowitz and Stegun 7.1.26: erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + p x),
// x >= 0, off by 1.5e-7 at most; in fp32 the function is within 3.0e-7 and GELU within 4.2e-7, which is what erff and its sum with 1
// lose too (4.5e-7).  Below 0, where that sum cancels, the error here falls with exp(-x^2) (g = -5: -1.4355e-6 for -1.4332e-6,
// with erff -1.4901e-6).  Gated bf16 4096 x 512 x 4096 38.2 -> 35.0 us, int8 1378 x 144 x 13968 45.4 -> 39.0.
#pragma once

#include <stdint.h>

#include "../../include/clpeak_b200_kernels.h"

namespace clpk {

__device__ __forceinline__ float exp_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float sigmoid(float x) { return rcp_approx(1.0f + exp_approx(-x)); }

constexpr float kGeluC = 0.7978845608028654f;       // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

// (1 + erf(g / sqrt(2))) / 2, and exp(-g^2 / 2)
__device__ __forceinline__ float normal_cdf(float g, float &e)
{
    const float x = fabsf(g) * 0.7071067811865476f, t = rcp_approx(1.0f + 0.3275911f * x);
    e = exp_approx(-0.5f * g * g);
    const float q = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
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
        return g < 0.0f ? 0.0f : g;                                 // a NaN stays one
    else
        return sigmoid(g);
}

// act(g) and act'(g)
template <int ACT>
__device__ __forceinline__ void activate_both(float g, float &a, float &da)
{
    if constexpr (ACT == CLPK_ACT_SILU) {
        const float p = sigmoid(g);
        a = g * p;
        da = p * (1.0f + g * (1.0f - p));
    } else if constexpr (ACT == CLPK_ACT_GELU_TANH) {
        const float c = fminf(fmaxf(g, -30.0f), 30.0f);             // beyond, p is 0 or 1 and the second term 0, whatever its factors
        const float p = sigmoid(2.0f * kGeluC * c * (1.0f + kGeluCubic * c * c));
        a = g * p;
        da = p + c * p * (1.0f - p) * (2.0f * kGeluC) * (1.0f + 3.0f * kGeluCubic * c * c);
    } else if constexpr (ACT == CLPK_ACT_GELU) {
        float e;
        const float cdf = normal_cdf(g, e);
        a = g * cdf;
        da = cdf + g * e * 0.3989422804014327f;                     // 1 / sqrt(2 pi)
    } else if constexpr (ACT == CLPK_ACT_RELU) {
        a = g < 0.0f ? 0.0f : g;
        da = g > 0.0f ? 1.0f : 0.0f;
    } else {
        const float p = sigmoid(g);
        a = p;
        da = p * (1.0f - p);
    }
}

} // namespace clpk
