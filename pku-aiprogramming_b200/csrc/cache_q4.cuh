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

// The smallest code whose scale s has 7.5 s >= top, and eight times that scale; `top` finite or infinite.  7.5 s is 0.9375 times half(c << 7),
// exactly (four bits times four), so a candidate is compared as it is.  The candidate: top / 0.9375 rounded up to four significant bits.
// The constant is the float below 16 / 15, so a quotient up to a scale does not come out above that scale, and one above it perhaps not above
// it either: a candidate is too small by one then, never too large.
__device__ __forceinline__ int q4_code(float top, float* scale8) {
    const float u = top * 1.0666666f;
    int c;
    float b;
    if (u < 6.103515625e-5f) {   // steps of 2^-17 below 2^-14
        c = (int)ceilf(u * 131072.f);
        b = (float)c * (1.f / 131072);
        if (0.9375f * b < top) b = (float)++c * (1.f / 131072);
    } else {
        unsigned bits = min((__float_as_uint(u) + 0xfffffu) >> 20, (unsigned)kQ4Top + 896);
        if (bits < kQ4Top + 896u && 0.9375f * __uint_as_float(bits << 20) < top) ++bits;
        c = (int)bits - 896;
        b = __uint_as_float(bits << 20);
    }
    *scale8 = b;
    return c;
}
__device__ __forceinline__ float q4_reciprocal(float x) {   // to a unit in the last place or so
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x / s to the nearest integer, ties to even, held to -8 .. 7, as the bits of 1.5 2^23 plus that: `inv` is 1 / s to 2^-22 or better (0 for s = 0).
constexpr uint32_t kQ4Bits = 0x4b400000u;   // of 1.5 2^23
// bf16 x: X 2^c / M with X of eight bits and M of four is either half-way between two integers or at least 2^-5 / 15 away from that, so the quotient
// is rounded to 2^-10 first, which puts the half-way ones where they belong and lets no other cross.
__device__ __forceinline__ uint32_t q4_level_bf16(float x, float inv) { return __float_as_uint(fminf(fmaf(x, inv, 12288.f), 12295.f) + (12582912.f - 12288.f)); }
// float x, `inv` the float nearest to 1 / s.  A quotient that is not half-way between two integers is rounded as it should be: half-way is h s with
// h s of eight bits, x is at least an ulp away from that, relatively 2^-24 (1 + 2^-8) or more, and inv is off by less than 2^-24 -- or by nothing,
// where h s is a power of two, below which floats are denser.  Half-way ones may go either way; the remainder x - r s is exact and says.
__device__ __forceinline__ uint32_t q4_level_f32(float x, float s, float inv) {
    float t = fmaf(x, inv, 12582912.f);
    const float rem = fmaf(12582912.f - t, s, x);
    if (fabsf(rem) == 0.5f * s && (__float_as_uint(t) & 1)) t += copysignf(1.f, rem);
    return __float_as_uint(fminf(t, 12582919.f));
}

}  // namespace ttk
