// Activations of the fused linear and gated epilogues and their derivatives, fp32, two elements at a time: products and
// sums as packed f32x2 instructions, exponential and reciprocal as the hardware's approximations.  Relative to itself a
// value is off by at most 2^-15, most of it the rounding of the exponential's argument far from zero, and so is each of the
// two terms of a slope: a bf16 result is rounded by 2^-8.  Values below about 1e-36, where the exponential or its
// reciprocal leaves the normal numbers, become zero.  A tile's epilogue evaluates 32768 of them per SM beside the tensor
// cores, so their instructions count.
#pragma once
#include <cuda_runtime.h>
#include "w8a8_arith.cuh"

namespace w8a8 {

// matches the order of the names in torch_ext.cpp and the DSV4_ACT_* constants
enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

constexpr float kInvSqrt2Pi = 0.39894228f;
constexpr float kGeluTanhC = 1.59576912f;   // 2 * sqrt(2 / pi): 0.5 * (1 + tanh(a)) = sigmoid(2 a)
constexpr float kGeluCubic = 0.044715f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / (1 + exp(-a z)) for a constant a
__device__ __forceinline__ float2 sigmoid2(float2 z, float a) {
    const float2 t = __fmul2_rn(z, splat2(-a * kLog2e));
    const float2 d = __fadd2_rn(make_float2(exp2_fast(t.x), exp2_fast(t.y)), splat2(1.0f));
    return make_float2(rcp_fast(d.x), rcp_fast(d.y));
}

// Phi(z), the normal distribution function, and e = exp(-z^2 / 2), which Phi's formula needs anyway and the density is
// made of.  1 - Phi(|z|) = 0.5 * erfc(x) = exp(-x^2) * 0.5 * erfcx(x), x = |z| / sqrt 2, with 0.5 * erfcx as t times a
// polynomial of degree six in t = 1 / (1 + 0.37339598 x) (the form of Hastings' approximations).  Constant and coefficients
// were fitted here to the smallest largest relative error on 0 <= x <= 9.5, a linear program over them: 4.9e-7, 9e-7 with
// fp32's roundings.  It is the relative error that counts: GELU far below zero is z times the tail, and a polynomial with an
// absolute bound (0.75e-7) was off by 3.6e-3 of the value at -6, about what bf16 rounds.  erfcf is exact to the last bits
// but takes four times the instructions and branches on its argument, which made the drain of a 7168-deep tile longer than
// its tensor-core work.
__device__ __forceinline__ float2 normal_cdf2(float2 z, float2& e) {
    const float2 a = make_float2(fabsf(z.x), fabsf(z.y));
    const float2 d = __ffma2_rn(a, splat2(0.26403083f), splat2(1.0f));
    const float2 t = make_float2(rcp_fast(d.x), rcp_fast(d.y));
    const float2 s = __fmul2_rn(__fmul2_rn(z, z), splat2(-0.5f * kLog2e));
    e = make_float2(exp2_fast(s.x), exp2_fast(s.y));
    float2 q = __ffma2_rn(t, splat2(-0.0693054696f), splat2(0.203423122f));
    q = __ffma2_rn(t, q, splat2(-0.0763239056f));
    q = __ffma2_rn(t, q, splat2(0.148744691f));
    q = __ffma2_rn(t, q, splat2(0.0804328837f));
    q = __ffma2_rn(t, q, splat2(0.107843366f));
    q = __ffma2_rn(t, q, splat2(0.105185018f));
    q = __fmul2_rn(__fmul2_rn(q, t), e);
    return make_float2(z.x > 0.0f ? 1.0f - q.x : q.x, z.y > 0.0f ? 1.0f - q.y : q.y);
}

__device__ __forceinline__ float relu(float z) { return z > 0.0f ? z : (z != z ? z : 0.0f); }   // a NaN stays one

template <int ACT>
__device__ __forceinline__ float2 act_value2(float2 z) {
    if constexpr (ACT == kActRelu) return make_float2(relu(z.x), relu(z.y));
    if constexpr (ACT == kActGelu) {
        float2 e;
        return __fmul2_rn(z, normal_cdf2(z, e));
    }
    if constexpr (ACT == kActGeluTanh) {
        const float2 c = __ffma2_rn(__fmul2_rn(__fmul2_rn(z, z), splat2(kGeluCubic)), z, z);
        return __fmul2_rn(z, sigmoid2(c, kGeluTanhC));
    }
    if constexpr (ACT == kActSilu) return __fmul2_rn(z, sigmoid2(z, 1.0f));
    return z;
}

// values, and the derivatives in `slope`
template <int ACT>
__device__ __forceinline__ float2 act_value_slope2(float2 z, float2& slope) {
    if constexpr (ACT == kActRelu) {
        slope = make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
        return act_value2<kActRelu>(z);
    }
    if constexpr (ACT == kActGelu) {
        float2 e;
        const float2 p = normal_cdf2(z, e);
        slope = __ffma2_rn(__fmul2_rn(z, splat2(kInvSqrt2Pi)), e, p);
        return __fmul2_rn(z, p);
    }
    if constexpr (ACT == kActGeluTanh || ACT == kActSilu) {
        // d(z sigmoid(c)) = p + z p (1 - p) c', with c' = 1 for SiLU
        float2 z2 = __fmul2_rn(z, z);
        z2 = make_float2(fminf(z2.x, 1e30f), fminf(z2.y, 1e30f));   // finite: 1 - p is zero long before
        const bool tanh_form = ACT == kActGeluTanh;
        const float2 p = tanh_form ? sigmoid2(__ffma2_rn(__fmul2_rn(z2, splat2(kGeluCubic)), z, z), kGeluTanhC) : sigmoid2(z, 1.0f);
        const float2 v = __fmul2_rn(z, p);
        float2 w = __ffma2_rn(p, splat2(-1.0f), splat2(1.0f));
        if (tanh_form) w = __fmul2_rn(w, __ffma2_rn(z2, splat2(3.0f * kGeluCubic * kGeluTanhC), splat2(kGeluTanhC)));
        slope = __ffma2_rn(v, w, p);
        return v;
    }
    slope = splat2(1.0f);
    return z;
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
