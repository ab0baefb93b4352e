// The number format of the 8-bit key/value cache: values are e4m3 codes times a power of two 2^e that 16 tokens of a head share, held as the
// byte e + 64, e of -40 .. 40.
//
// Why these: a floating code loses nothing by a coarse scale -- its relative error is 2^-4 wherever it is normal, 2^-6 .. 448 of the scale -- so a power of
// two serves as well as a finer one, and a block whose tokens come one after the other can be moved to a larger exponent with its normal values
// unchanged.  Codes are exact in half, code times 2^e in bf16.  The exponent's range leaves a sum of probabilities over 2^e room in 32 bits on either side.
#pragma once
#include <cuda_fp16.h>

#include "common.h"

namespace ttk {

constexpr int kQ8Low = -40, kQ8High = 40, kQ8Bias = 64, kQ8Block = 16;

__host__ __device__ constexpr long long q8_page_bytes(int page, int D) { return (long long)page * D + (page / kQ8Block + 31) / 32 * 32; }
__device__ __forceinline__ int q8_exponent(int byte) { return min(max(byte - kQ8Bias, kQ8Low), kQ8High); }
__device__ __forceinline__ float q8_power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// The smallest exponent with 448 2^e >= the finite value of these bits (448 is 1.75 2^8)
__device__ __forceinline__ int q8_exponent_of(unsigned bits) {
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(e, kQ8Low), kQ8High);
}
__device__ __forceinline__ uint32_t q8_encode4(float a, float b, float c, float d) {   // four codes, the first lowest; beyond 448, infinities too: 448
    uint32_t w;
    asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\nmov.b32 %0, {lo, hi};\n}" : "=r"(w) : "f"(a), "f"(b), "f"(c), "f"(d));
    return w;
}
// Four codes as halves: the lower two, the upper two.  (The header's conversion of two takes 6.5 cycles of an SM's quarter, this one two.)
__device__ __forceinline__ void q8_halves(uint32_t w, uint32_t& lower, uint32_t& upper) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}" : "=r"(lower), "=r"(upper) : "r"(w));
}
__device__ __forceinline__ void q8_floats(uint32_t w, float (&f)[4]) {
    uint32_t h[2];
    q8_halves(w, h[0], h[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        f[2 * i] = two.x;
        f[2 * i + 1] = two.y;
    }
}

}  // namespace ttk
