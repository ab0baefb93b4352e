// What the kernels that turn heads by their positions share: values and vectors of a type, the sine and cosine of a pair, and
// where a CTA's tokens are.
#pragma once
#include "common.h"

namespace ttk {

template <typename T> __device__ __forceinline__ float rt_get(T v);
template <> __device__ __forceinline__ float rt_get(float v) { return v; }
template <> __device__ __forceinline__ float rt_get(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T rt_put(float v);
template <> __device__ __forceinline__ float rt_put(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 rt_put(float v) { return __float2bfloat16_rn(v); }

template <typename T, int kV> struct alignas(sizeof(T) * kV) RtVec { T v[kV]; };

// scale * (cos, sin) of position p times frequency f, the sine's sign turned round with `back`.  In 32 bits a position of 10^6 leaves 0.03 of a
// radian of the product, so it is taken in 64, in turns, less its nearest whole number; the rest, at most half a turn, goes through sincospif.
__device__ __forceinline__ float2 rt_turn(int p, double f, float scale, int back) {
    const double turns = (double)p * f * 0.15915494309189533576888;   // / 2 pi
    float sn, co;
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &co);
    return make_float2(scale * co, back ? -scale * sn : scale * sn);
}

// Batch entry and row of the tokens that follow t0, without a division for each.
struct RtPlaces {
    unsigned t0, b0, S;
    __device__ __forceinline__ RtPlaces(unsigned first, int B, int rows) : t0(first), b0(B > 1 ? first / (unsigned)rows : 0), S((unsigned)rows) {}
    __device__ __forceinline__ void at(int t, int* b, int* s) const {
        unsigned x = t0 - b0 * S + t, y = b0;
        while (x >= S) {
            x -= S;
            ++y;
        }
        *b = (int)y;
        *s = (int)x;
    }
};

}  // namespace ttk
