// Activations of the fused linear and gated epilogues and their derivatives, fp32.  They take CUDA's fast exponential and
// reciprocal, whose relative error (about 2^-21 at the arguments where the result still matters) is far below the bf16
// step of every output that they reach.
#pragma once
#include <cuda_runtime.h>

namespace w8a8 {

// matches the order of the names in torch_ext.cpp and the DSV4_ACT_* constants
enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

constexpr float kSqrtHalf = 0.70710678f;
constexpr float kInvSqrt2Pi = 0.39894228f;
constexpr float kGeluTanhC = 1.59576912f;   // 2 * sqrt(2 / pi): 0.5 * (1 + tanh(a)) = sigmoid(2 a)
constexpr float kGeluCubic = 0.044715f;

__device__ __forceinline__ float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// Phi(z), the normal distribution function, and exp(-z^2 / 2), which Phi's formula needs anyway and the density is made of.
// 0.5 * erfc(|z| / sqrt 2) by Abramowitz and Stegun, Handbook of Mathematical Functions, formula 7.1.26: a polynomial of
// degree five in 1 / (1 + 0.3275911 x) times exp(-x^2), off by at most 0.75e-7.  erfcf is exact to the last bits but takes
// four times the instructions and branches on its argument, which made the drain of a 7168-deep tile longer than its
// tensor-core work.
__device__ __forceinline__ float2 normal_cdf_exp(float z) {
    const float x = fabsf(z) * kSqrtHalf;
    const float t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f));
    const float e = __expf(-x * x);
    float q = fmaf(t, 1.061405429f, -1.453152027f);
    q = fmaf(t, q, 1.421413741f);
    q = fmaf(t, q, -0.284496736f);
    q = fmaf(t, q, 0.254829592f);
    q = q * t * e * 0.5f;
    return make_float2(z > 0.0f ? 1.0f - q : q, e);
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == kActRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if constexpr (ACT == kActGelu) return z * normal_cdf_exp(z).x;
    if constexpr (ACT == kActGeluTanh) return z * sigmoid_fast(kGeluTanhC * fmaf(kGeluCubic * z * z, z, z));
    if constexpr (ACT == kActSilu) return z * sigmoid_fast(z);
    return z;
}

// value and derivative together
template <int ACT>
__device__ __forceinline__ float2 act_value_slope(float z) {
    if constexpr (ACT == kActRelu) return make_float2(act_value<kActRelu>(z), z > 0.0f ? 1.0f : 0.0f);
    if constexpr (ACT == kActGelu) {
        const float2 p = normal_cdf_exp(z);
        return make_float2(z * p.x, fmaf(z * kInvSqrt2Pi, p.y, p.x));
    }
    if constexpr (ACT == kActGeluTanh) {
        const float z2 = z * z;
        const float p = sigmoid_fast(kGeluTanhC * fmaf(kGeluCubic * z2, z, z));
        return make_float2(z * p, fmaf(z * p * (1.0f - p), kGeluTanhC * fmaf(3.0f * kGeluCubic, z2, 1.0f), p));
    }
    if constexpr (ACT == kActSilu) {
        const float p = sigmoid_fast(z);
        return make_float2(z * p, fmaf(z * p, 1.0f - p, p));
    }
    return make_float2(z, 1.0f);
}

template <int V>
struct ActConst { static constexpr int value = V; };

// f(ActConst<act>{}): the choice is uniform over the launch, so one branch per call
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
        case kActRelu: f(ActConst<kActRelu>{}); break;
        case kActGelu: f(ActConst<kActGelu>{}); break;
        case kActGeluTanh: f(ActConst<kActGeluTanh>{}); break;
        case kActSilu: f(ActConst<kActSilu>{}); break;
        default: f(ActConst<kActNone>{}); break;
    }
}

}  // namespace w8a8
