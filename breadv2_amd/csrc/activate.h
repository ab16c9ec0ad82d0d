// activate.h — the activations of the products' epilogues (BREAD_ACT_*).
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/bread_moe.h"

// 1 / (1 + exp(-v)): 1 and 0 far out
__device__ __forceinline__ float sigmoid(float v)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}

// The activations to a few 2^-24 of v.  GELU by Abramowitz and Stegun 7.1.26, erfc(x) = exp(-x^2) times a
// polynomial of 1 / (1 + 0.3275911 x) to 1.5e-7: a third of the library erf's instructions.
__device__ __forceinline__ float activate(float v, int act)
{
    switch (act) {
    case BREAD_ACT_SILU: return v * sigmoid(v);
    case BREAD_ACT_GELU: {
        const float x = fabsf(v) * 0.70710678f;
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
        float p = fmaf(1.061405429f, t, -1.453152027f);
        p = fmaf(p, t, 1.421413741f);
        p = fmaf(p, t, -0.284496736f);
        p = fmaf(p, t, 0.254829592f);
        const float half = 0.5f * p * t * __builtin_amdgcn_exp2f(-1.44269504f * x * x);  // erfc(x) / 2
        return v * (v < 0.f ? half : 1.0f - half);
    }
    case BREAD_ACT_GELU_TANH: return v * sigmoid(1.59576912f * (v + 0.044715f * v * v * v));
    case BREAD_ACT_RELU: return v < 0.f ? 0.f : v;  // NaN stays NaN
    }
    return v;
}
