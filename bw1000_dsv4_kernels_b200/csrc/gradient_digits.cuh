// The fixed-point form of a gradient row: v = rint(t / s) with s = top / 32639, cut into digits v = 256 hi + mid with hi in
// [-127, 127] and mid in [-128, 127] (32639 = 127 * 256 + 127 is the largest v whose digits are int8).  |t - s v| <= s / 2,
// 2^-16 of the row's largest magnitude `top`.
//
// For an element of the row's typical size (the square of the mean square root of its magnitudes, which a few outliers
// hardly move) that is at most 2^-8 of itself, as long as the typical size is at least top / 256.  Rows of gradients are
// mostly far above that: normally distributed ones at top / 7, dg and du of a gated projection at top / 30 to top / 160.
// A row below it, most of it far smaller than its outliers, is `wide` and has a third digit:
// v = rint(256 t / s) = 65536 hi + 256 mid + lo, |t - s v / 256| <= s / 512, 2^-24 of top.  With two digits, 600 normal
// elements beside one of 3000 times their size gave dx rows off by 2.7 % where the outlier meets zeros of the weight (a
// bf16 operand: 0.2 %, three digits: 0.01 %).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace w8a8 {

constexpr float kDigitMax = 32639.0f;
constexpr float kTopFloor = 1e-30f;   // rows of zeros (and of magnitudes below it, which become zeros)
constexpr float kWideRoot = 16.0f;    // a row whose typical size is less than top / 16^2 takes the third digit

// What a part of a row (a tile's columns, or all of them) says about the row's size: its largest magnitude, as the bits of
// a non-negative float (an integer maximum keeps a NaN, which then reaches the whole row of the result), and the sum of
// the square roots of its magnitudes, within 6 % (half of a float's bits, with the exponent's bias put right).
struct alignas(8) RowSize {
    unsigned top;
    float roots;
    static __device__ __forceinline__ RowSize none() { return {0u, 0.0f}; }
    __device__ __forceinline__ void add(float t) {
        const unsigned bits = __float_as_uint(t) & 0x7fffffffu;
        top = max(top, bits);
        roots = __fadd_rn(roots, __uint_as_float((bits >> 1) + 0x1fc00000u));
    }
    __device__ __forceinline__ void add(const float2& t) { add(t.x); add(t.y); }
    __device__ __forceinline__ void add(const RowSize& o) {
        top = max(top, o.top);
        roots = __fadd_rn(roots, o.roots);
    }
    // together with the lane `o` away; both get the same bits
    __device__ __forceinline__ void add_lane(int o) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        roots = __fadd_rn(roots, __shfl_xor_sync(0xffffffffu, roots, o));
    }
    // with share = kWideRoot / elements of the row; rows that hold an infinity or a NaN are not wide
    __device__ __forceinline__ bool wide(float share) const {
        const float t = __uint_as_float(top), root = __fmul_rn(roots, share);
        return t >= kTopFloor && top < 0x7f800000u && __fmul_rn(root, root) < t;
    }
};

// A row's size as the gradient product takes it: the bits of `top`, and whether the row is wide in the bit of its sign.
__device__ __forceinline__ unsigned packed_size(unsigned top, bool wide) { return wide ? top | 0x80000000u : top; }
__device__ __forceinline__ bool is_wide(unsigned size) { return (size >> 31) != 0; }
__device__ __forceinline__ float top_of_size(unsigned size) { return __uint_as_float(size & 0x7fffffffu); }

__device__ __forceinline__ float digit_scale(float top) { return __fdiv_rn(top < kTopFloor ? kTopFloor : top, kDigitMax); }
__device__ __forceinline__ float digit_inverse(float top) { return __fdiv_rn(kDigitMax, top < kTopFloor ? kTopFloor : top); }

// Digits of a row's elements: t -> w + 0x8080, w = 65536 hi + 256 mid + lo the value in three digits, whose lowest is zero
// unless the row is wide.  The bytes of that sum are hi, mid + 128 and lo + 128 (mod 256): a carry into the digit above is
// what makes the one below signed.  |w| <= 32639 * 256 + 2 (the products are off by 2^-22 of themselves), so hi is at most 127.
struct RowDigits {
    float inv;
    int shift;
    static __device__ __forceinline__ RowDigits make(unsigned top, bool wide) {
        return {__fmul_rn(digit_inverse(__uint_as_float(top)), wide ? 256.0f : 1.0f), wide ? 0 : 8};
    }
    __device__ __forceinline__ unsigned of(float t) const { return ((unsigned)__float2int_rn(__fmul_rn(t, inv)) << shift) + 0x8080u; }
};
// digit 2 (hi), 1 (mid) or 0 (lo) of four elements
template <int DIGIT>
__device__ __forceinline__ uint32_t pack_digit(const unsigned (&w)[4]) {
    constexpr unsigned kPick = DIGIT | ((4 + DIGIT) << 4);
    const uint32_t v = __byte_perm(__byte_perm(w[0], w[1], kPick), __byte_perm(w[2], w[3], kPick), 0x5410);
    return DIGIT == 2 ? v : v ^ 0x80808080u;
}

// 256 hi + mid of two exact int32 sums: each rounds to fp32 once, the product with 256 does not round
__device__ __forceinline__ float digit_sum(int hi, int mid) { return __fmaf_rn(__int2float_rn(hi), 256.0f, __int2float_rn(mid)); }
// ... and lo / 256 more
__device__ __forceinline__ float wide_digit_sum(float sum, int lo) { return __fmaf_rn(__int2float_rn(lo), 1.0f / 256.0f, sum); }

}  // namespace w8a8
