// Activations of a gated feed-forward layer and their derivatives, in fp32.
//
// exp is ex2.approx behind a multiplication (__expf): its relative error grows with |x| to 5e-6 at |x| = 88, where the sigmoid
// it stands in has long been 0 or 1; below |x| = 8 it is under 5e-7.  The results are rounded to 16 bits almost everywhere
// they are used.  tanh-GELU is a sigmoid too: (1 + tanh y) / 2 = 1 / (1 + exp(-2 y)).
#pragma once

#include <stdint.h>

#include "../../include/clpeak_b200_kernels.h"

namespace clpk {

// __fdividef gives 0 for a divisor beyond 2^126, which is what the sigmoid rounds to there
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

constexpr float kGeluC = 0.7978845608028654f;       // sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

template <int ACT>
__device__ __forceinline__ float activate(float g)
{
    if constexpr (ACT == CLPK_ACT_SILU)
        return __fdividef(g, 1.0f + __expf(-g));
    else if constexpr (ACT == CLPK_ACT_GELU_TANH)
        return __fdividef(g, 1.0f + __expf(-2.0f * kGeluC * (g + kGeluCubic * g * g * g)));
    else if constexpr (ACT == CLPK_ACT_GELU)
        return 0.5f * g * (1.0f + erff(g * 0.7071067811865476f));
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
        const float p = sigmoid(2.0f * kGeluC * (c + kGeluCubic * c * c * c));
        a = g * p;
        da = p + c * p * (1.0f - p) * (2.0f * kGeluC) * (1.0f + 3.0f * kGeluCubic * c * c);
    } else if constexpr (ACT == CLPK_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.7071067811865476f));
        a = g * cdf;
        da = cdf + g * __expf(-0.5f * g * g) * 0.3989422804014327f; // 1 / sqrt(2 pi)
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
