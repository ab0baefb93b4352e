// The number format of the 4-bit key/value cache: 32 channels share a scale code c, a value is (n - 8) s with n in 0 .. 15 and
// s = half(c << 7) / 8, an unsigned float of five exponent and three mantissa bits.
//
// Why these: a scale of four significant bits times an integer of four has eight, so a value is exact in bf16 and in half, the
// unpacked operand of a tensor-core product needs no rounding, and c << 7 is the scale's own bit pattern.  The largest
// code written is 222 (896 = 7 * 128): 9 * 8 s then still is a finite half, which lets one fused multiply-add unpack and scale.
// Against a scale of 16 bits the step is 6 % larger on average; it takes 0.25 bits a value instead of 0.5.
#pragma once
#include <cuda_fp16.h>

#include "common.h"

namespace ttk {

constexpr int kQ4Top = 222, kQ4NaN = 255;

__host__ __device__ constexpr int q4_row_bytes(int D) { return D / 2 + D / 32; }
// half(code << 7): eight times the scale
__device__ __forceinline__ float q4_scale8(int code) { return __half2float(__ushort_as_half((unsigned short)(code << 7))); }

// The smallest code whose scale s has 7.5 s >= top (0.9375 times half(c << 7)); `top` finite or infinite.  The product is exact: four bits
// times four.
__device__ __forceinline__ int q4_code(float top) {
    const float u = top * 1.0666666667f;   // top / 0.9375 up to a rounding: the right code or a neighbour
    const unsigned b = __float_as_uint(u);
    // round up to four significant bits; below 2^-14 in steps of 2^-17
    int c = u < 6.103515625e-5f ? (int)ceilf(u * 131072.f) : (int)min((b + 0xfffffu) >> 20, 2047u) - 896;
    if (c < kQ4Top && 0.9375f * q4_scale8(c) < top) ++c;
    if (c > 0 && c <= kQ4Top && 0.9375f * q4_scale8(c - 1) >= top) --c;
    return min(c, kQ4Top);
}
// x / s to the nearest integer, ties to even, held to -8 .. 7, plus 8.  `inv` is 1 / s (0 for s = 0) to a rounding, which leaves the
// quotient's nearest integer or the next one; the remainder x - r s is exact (s has four bits, r at most five) and decides.
__device__ __forceinline__ unsigned q4_level(float x, float s, float inv) {
    float r = rintf(x * inv);
    const float rem = fmaf(-r, s, x), far = fabsf(rem), half_step = 0.5f * s;
    if (far > half_step || (far == half_step && s > 0.f && ((int)fminf(fabsf(r), 64.f) & 1))) r += copysignf(1.f, rem);
    return (unsigned)((int)fminf(fmaxf(r, -8.f), 7.f) + 8);
}

}  // namespace ttk
