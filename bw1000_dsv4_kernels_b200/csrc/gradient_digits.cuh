// The fixed-point form of a gradient row: v = rint(t / s) with s = top / 32639, cut into digits v = 256 hi + lo with hi in
// [-127, 127] and lo in [-128, 127] (32639 = 127 * 256 + 127 is the largest v whose digits are int8).  |t - s v| <= s / 2,
// 2^-16 of the row's largest magnitude.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace w8a8 {

constexpr float kDigitMax = 32639.0f;
constexpr float kTopFloor = 1e-30f;   // rows of zeros (and of magnitudes below it, which become zeros)

__device__ __forceinline__ float digit_scale(float top) { return __fdiv_rn(top < kTopFloor ? kTopFloor : top, kDigitMax); }
__device__ __forceinline__ float digit_inverse(float top) { return __fdiv_rn(kDigitMax, top < kTopFloor ? kTopFloor : top); }

__device__ __forceinline__ int digits_of(float t, float inv) {
    // |t * inv| <= 32639 (1 + 2^-22): the rounded value stays within the digits' range
    return __float2int_rn(__fmul_rn(t, inv));
}
__device__ __forceinline__ int digit_hi(int v) { return (v + 128) >> 8; }
__device__ __forceinline__ int digit_lo(int v) { return v - (digit_hi(v) << 8); }

// s * (256 hi + lo) of two exact int32 sums: each rounds to fp32 once, the product with 256 does not round
__device__ __forceinline__ float digit_value(int hi, int lo, float s) {
    return __fmul_rn(__fmaf_rn(__int2float_rn(hi), 256.0f, __int2float_rn(lo)), s);
}

}  // namespace w8a8
