// Rotary positions on query and key heads, several axes, forward and backward.
//
// Pair i of a token turns by p[axis_i] * f_i (rt_turn).
//
// HBM-bound: every value is read and written once.  A CTA takes a few tokens: their R / 2 sines and cosines go to shared memory
// once (for up to 40 heads that use them), then a thread keeps its place in the head -- up to 16 bytes of one half and their partners
// in the other, or of neighbours -- and walks over tokens and heads, so an access of a warp is whole rows.
#include "rotary_parts.cuh"

namespace ttk {

constexpr int kRotaryThreads = 256;

// A token's rows of one of the two tensors: of head 0 in the input and the output.
template <typename T> struct alignas(16) RtRows {
    const T* x;
    T* y;
};

// kV values per access.  A unit of work is `kV` pairs in halves, or kV / 2 neighbouring pairs (one pair at kV = 1), or `copied`
// bytes of the channels behind R; blockDim = {units per head, rows at a time}.
template <typename T, int kV, bool kNeighbours>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a, int tokens_per_cta, int turned, int copied, float per_half) {
    using Vec = RtVec<T, kV>;
    constexpr int kPairs = kNeighbours && kV > 1 ? kV / 2 : kV;   // of a unit
    extern __shared__ float4 sm[];
    RtRows<T>* rows = reinterpret_cast<RtRows<T>*>(sm);   // [tokens_per_cta][2]
    // [tokens_per_cta][R / 2] scale * (cos, sin), two pairs of a unit beside each other and then the same two of the next unit, so that what a
    // warp reads at a time is whole banks
    float2* cs = reinterpret_cast<float2*>(rows + 2 * tokens_per_cta);
    const int half = a.R / 2, tid = threadIdx.y * blockDim.x + threadIdx.x, n_threads = blockDim.x * blockDim.y;
    const unsigned t0 = blockIdx.x * (unsigned)tokens_per_cta, n_tok = (unsigned)a.B * (unsigned)a.S;
    const int here = (int)min((unsigned)tokens_per_cta, n_tok - t0);
    const RtPlaces places(t0, a.B, a.S);
    grid_let_next_start();
    grid_wait_for_previous();
    for (int i = tid; i < here * half; i += n_threads) {
        const int t = (int)(((float)i + 0.5f) * per_half), pair = i - t * half;   // i < 2^13: exact
        int b, s;
        places.at(t, &b, &s);
        const int axis = a.axes ? min(max(a.axes[pair], 0), a.n_axes - 1) : 0;
        const int p = a.pos[axis * a.pos_axis + b * a.pos_batch + s];
        const int u = pair / kPairs, e = pair % kPairs;
        cs[t * half + (kPairs == 1 ? u : 2 * ((e >> 1) * turned + u) + (e & 1))] = rt_turn(p, a.inv_freq[pair], a.scale, a.back);
    }
    for (int i = n_threads - 1 - tid; i < 2 * here; i += n_threads) {
        int b, s;
        places.at(i >> 1, &b, &s);
        const int w = i & 1;
        rows[i] = RtRows<T>{(const T*)a.x[w] + b * a.xs[w][0] + s * a.xs[w][2], (T*)a.y[w] + b * a.ys[w][0] + s * a.ys[w][2]};
    }
    __syncthreads();
    const int u = threadIdx.x, heads = a.heads[0] + a.heads[1];
    const bool turn = u < turned;
    // the unit's channels: kV at c0, and in halves their partners at c1; or `copied` bytes behind R
    const int c0 = kNeighbours && kV == 1 ? 2 * u : u * kV, copy_at = (u - turned) * copied;
    const int c1 = kNeighbours ? c0 + 1 : c0 + half;
    const bool two = turn && (!kNeighbours || kV == 1);
    int t = 0, h = threadIdx.y;
    while (h >= heads) {
        h -= heads;
        ++t;
    }
    while (t < here) {
        const bool second = h >= a.heads[0];
        const int head = second ? h - a.heads[0] : h;
        const RtRows<T> r = rows[2 * t + second];
        const T* x = r.x + head * (second ? a.xs[1][1] : a.xs[0][1]);
        T* y = r.y + head * (second ? a.ys[1][1] : a.ys[0][1]);
        if (turn) {
            Vec v0 = *reinterpret_cast<const Vec*>(x + c0), v1;
            if (two) v1 = *reinterpret_cast<const Vec*>(x + c1);
            const float2* from = cs + t * half + (kPairs == 1 ? u : 2 * u);
            float2 f[kPairs];
            if (kPairs == 1) {
                f[0] = *from;
            } else {
#pragma unroll
                for (int e = 0; e < kPairs; e += 2) {
                    const float4 z = *reinterpret_cast<const float4*>(from + e * turned);
                    f[e] = make_float2(z.x, z.y);
                    f[(e + 1) % kPairs] = make_float2(z.z, z.w);
                }
            }
            if (two) {
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    const float x1 = rt_get(v0.v[e]), x2 = rt_get(v1.v[e]);
                    v0.v[e] = rt_put<T>(x1 * f[e % kPairs].x - x2 * f[e % kPairs].y);
                    v1.v[e] = rt_put<T>(x2 * f[e % kPairs].x + x1 * f[e % kPairs].y);
                }
                *reinterpret_cast<Vec*>(y + c1) = v1;
            } else {
#pragma unroll
                for (int e = 0; e + 1 < kV; e += 2) {
                    const float x1 = rt_get(v0.v[e]), x2 = rt_get(v0.v[e + 1]);
                    v0.v[e] = rt_put<T>(x1 * f[e / 2].x - x2 * f[e / 2].y);
                    v0.v[e + 1] = rt_put<T>(x2 * f[e / 2].x + x1 * f[e / 2].y);
                }
            }
            *reinterpret_cast<Vec*>(y + c0) = v0;
        } else if (x != y) {
            const char* from = reinterpret_cast<const char*>(x + a.R) + copy_at;
            char* to = reinterpret_cast<char*>(y + a.R) + copy_at;
            if (copied == 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
            else if (copied == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
            else if (copied == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
            else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
        }
        h += blockDim.y;
        while (h >= heads) {
            h -= heads;
            ++t;
        }
    }
}

template <typename T, int kV, bool kNeighbours>
static cudaError_t launch_rotary(const RotaryArgs& a, int aligned, cudaStream_t st) {
    const int behind = (a.D - a.R) * (int)sizeof(T);
    int copied = aligned;   // the widest copies that begin and end where these channels do
    while ((a.R * (int)sizeof(T)) % copied || behind % copied) copied /= 2;
    const int turned = kNeighbours ? (kV == 1 ? a.R / 2 : a.R / kV) : a.R / 2 / kV, units = turned + behind / copied;
    const dim3 block(units, kRotaryThreads / units);
    const long long n_tok = (long long)a.B * a.S, heads = a.heads[0] + a.heads[1];
    // Tokens per CTA: up to four units per thread, the sines of one CTA run under the rows of others; fewer where all CTAs are resident at once then (eight
    // per SM), and more, up to half as many again, where that leaves no second wave.  With inputs from memory, us at 2 / 3 / 4 / 5 / 7 / 9 tokens: 4096 tokens
    // of 16 heads of 64 floats 9.7 / 11.8 / 8.5 / 9.9 / 12.2 / 15.3 (4 are one wave); 5000 of 20 heads of 80 bf16 8.7 / 9.7 / 9.4 / 7.7 / 10.0 / 11.7 (5 are);
    // 8192 of 9 heads of 128 9.9 / 8.6 / 8.9 / 8.9 / 7.9 / 9.6 (7 are); 16384 of 40 heads of 128 53.3 / 53.6 / 53.9 / 55.2 / 56.8 / 58.3, 6.3 TB/s.  Few tokens and
    // heads are bound by the sines: 15240 tokens of three heads, R = 256: 14 where the rows take 7.3.  (Two rows loaded ahead of the sines, 80 registers: 85 us for
    // 58.  Angles as products of 64-bit integers: 0.5 us slower, but 12.5 for 13.6 with three heads.)
    const long long resident = 8LL * sm_count(), one_wave = (n_tok + resident - 1) / resident;
    long long per = 4LL * block.y / heads;
    if (per > one_wave || 3 * per >= 2 * one_wave) per = one_wave;
    const size_t token = (size_t)a.R / 2 * sizeof(float2) + 2 * sizeof(RtRows<T>);
    const long long fits = 27 * 1024 / (long long)token;   // eight CTAs' on an SM; at most 128 pairs: 26 tokens
    if (per > fits) per = fits;
    if (per < 1) per = 1;
    LaunchScope ls(K_ROTARY, st);
    return launch_overlapped(rotary_kernel<T, kV, kNeighbours>, (unsigned)((n_tok + per - 1) / per), block, (size_t)per * token, st, a, (int)per, turned, copied,
                             2.f / (float)a.R);
}
// kV: the most values that can be turned at a time, from rows that lie at multiples of `aligned` bytes.  10,356 tokens of 40 heads of 80 bf16 channels,
// R = 20 and 40 in halves (2 and 4 values), 20.5 us of bytes: 53.5 and 37.4 us, 68.5 and 45.1 with copies as narrow, 88.9 and 92.0 with one value at
// a time.  Bound by the instructions per access.
template <typename T, int kV>
static cudaError_t launch_rotary_width(const RotaryArgs& a, int interleaved, int aligned, cudaStream_t st) {
    if constexpr (kV > 1) {
        if ((int)(kV * sizeof(T)) > aligned || (interleaved ? a.R : a.R / 2) % kV) return launch_rotary_width<T, kV / 2>(a, interleaved, aligned, st);
    }
    return interleaved ? launch_rotary<T, kV, true>(a, aligned, st) : launch_rotary<T, kV, false>(a, aligned, st);
}
template <typename T>
static cudaError_t launch_rotary_type(const RotaryArgs& a, int interleaved, cudaStream_t st) {
    unsigned long long places = 16;   // or-ed: the lowest bit set is what all are multiples of
    for (int i = 0; i < 2; ++i) {
        if (!a.heads[i]) continue;
        places |= (uintptr_t)a.x[i] | (uintptr_t)a.y[i];
        const int n[3] = {a.B, a.heads[i], a.S};
        for (int d = 0; d < 3; ++d)
            if (n[d] > 1) places |= (unsigned long long)(a.xs[i][d] | a.ys[i][d]) * sizeof(T);
    }
    return launch_rotary_width<T, 16 / sizeof(T)>(a, interleaved, (int)(places & (0 - places)), st);
}
cudaError_t rotary(const RotaryArgs& a, int bf16, int interleaved, cudaStream_t st) {
    return bf16 ? launch_rotary_type<__nv_bfloat16>(a, interleaved, st) : launch_rotary_type<float>(a, interleaved, st);
}

}  // namespace ttk
