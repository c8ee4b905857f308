// Activations of the fused linear and gated epilogues and their derivatives, fp32.  exp and erfc are CUDA's own; the
// sigmoid takes the fast exponential, whose relative error (about 2^-21 at the arguments where the result still
// matters) is far below the bf16 step of every output that it reaches.
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

// erfc(-z / sqrt 2) rather than 1 + erf: it keeps its relative accuracy where the normal distribution's tail is small
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f * erfcf(-z * kSqrtHalf); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == kActRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if constexpr (ACT == kActGelu) return z * normal_cdf(z);
    if constexpr (ACT == kActGeluTanh) return z * sigmoid_fast(kGeluTanhC * fmaf(kGeluCubic * z * z, z, z));
    if constexpr (ACT == kActSilu) return z * sigmoid_fast(z);
    return z;
}

// value and derivative together
template <int ACT>
__device__ __forceinline__ float2 act_value_slope(float z) {
    if constexpr (ACT == kActRelu) return make_float2(act_value<kActRelu>(z), z > 0.0f ? 1.0f : 0.0f);
    if constexpr (ACT == kActGelu) {
        const float p = normal_cdf(z);
        return make_float2(z * p, fmaf(z * kInvSqrt2Pi, __expf(-0.5f * z * z), p));
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
