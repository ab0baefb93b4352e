// The number format of the 8-bit key/value cache: values are e4m3 codes times a power of two 2^e that 16 tokens of a head share, held as the
// byte e + 64, e of -40 .. 40.
//
// Why these: a floating code loses nothing by a coarse scale -- its relative error is 2^-4 wherever it is normal, 2^-6 .. 448 of the scale -- so a power of
// two serves as well as a finer one, and a block whose tokens come one after the other can be moved to a larger exponent with its normal values
// unchanged.  Codes are exact in half, code times 2^e in bf16.  The exponent's range leaves a sum of probabilities over 2^e room in 32 bits on either side.
#pragma once
#include <cuda_fp8.h>

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
__device__ __forceinline__ uint32_t q8_encode2(float lo, float hi) {   // two codes, the second in bits 8 .. 15; beyond 448, infinities too: 448
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t q8_halves(uint32_t codes) {   // of the low 16 bits
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
    return h.x | (uint32_t)h.y << 16;
}

}  // namespace ttk
