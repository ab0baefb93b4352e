// Writing new keys and values into the 8-bit cache, and reading sequences back as packed bf16.
//
// Writing: a warp has the tokens of one call that go to one block of 16, of one head: it finds their largest value, and with the exponent that the
// block has from earlier tokens the new one, moves what is there where that grew, and writes the codes.  Tokens of a block lie next to each other in
// a call (a sequence's do), so the first of a run, whose predecessor goes elsewhere, stands for it, with up to 15 behind it.  Both directions are bound by HBM: D = 128 in bf16 is 256 bytes a
// token and head, its codes 128.
//
// Measured, 8 heads of 128 in bf16: writing 20,000 tokens 23.9 us, 5.2 TB/s; reading 61,000 back 61.3 us, 6.1 TB/s (a copy runs at 6.6); 64 single tokens, both calls, 6.5 us.
// Issue slots of writing are 55 % busy (the largest value, and the rounding, of each); reading waits for memory alone.
#include "cache_q8.cuh"
#include "sm100_ptx.cuh"

namespace ttk {

constexpr int kQ8Threads = 256, kQ8Most = 32;   // tokens that a CTA looks for runs in

// What a row of D values is to a warp: 16 bytes a lane, kRows rows at a time; a block's are kLoads loads of four registers.  kCtas: as many per SM as hold them; 20,000
// tokens of 8 heads, us with one CTA fewer and so: bf16 D = 128 24.3, 23.9 (4; 5 take 25.1), D = 64 16.0, 14.9 (5), floats D = 128 58.5, 41.8 (2), D = 64 26.0, 22.1 (3).
template <typename T, int D>
struct Q8Rows {
    static constexpr int kV = 16 / sizeof(T), kLanes = D / kV, kRows = 32 / kLanes, kLoads = kQ8Block / kRows;
    static constexpr int kCtas = sizeof(T) == 2 ? (D == 64 ? 5 : 4) : D == 64 ? 3 : 2;
};

// 16 bytes of them; 0 where there is no token.
template <typename T> struct Q8Values;
template <> struct Q8Values<__nv_bfloat16> {
    uint32_t w[4];
    template <bool kWide> __device__ __forceinline__ void load(const __nv_bfloat16* p, bool there) {
        if (!there) {
            w[0] = w[1] = w[2] = w[3] = 0;
        } else if (kWide) {
            const uint4 r = *reinterpret_cast<const uint4*>(p);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        } else {
            const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
    // magnitudes' bits, two in a word: ordered as the values, infinities and NaN above them
    __device__ __forceinline__ unsigned largest(unsigned top) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
        return top;
    }
    static __device__ __forceinline__ unsigned bits(unsigned top) { return max(top << 16, top & 0xffff0000u); }
};
template <> struct Q8Values<float> {
    float x[4];
    template <bool kWide> __device__ __forceinline__ void load(const float* p, bool there) {
        if (!there) {
            x[0] = x[1] = x[2] = x[3] = 0.f;
        } else if (kWide) {
            const float4 r = *reinterpret_cast<const float4*>(p);
            x[0] = r.x; x[1] = r.y; x[2] = r.z; x[3] = r.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = p[i];
        }
    }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
    __device__ __forceinline__ unsigned largest(unsigned top) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        return top;
    }
    static __device__ __forceinline__ unsigned bits(unsigned top) { return top; }
};

template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(kQ8Threads, Q8Rows<T, D>::kCtas) cache_append_q8_kernel(const T* __restrict__ k, const T* __restrict__ v, const int* __restrict__ slots, int n_tok, int tokens_per_cta,
                                                                     int hkv, long long k_tok, long long k_head, long long v_tok, long long v_head, unsigned char* kc,
                                                                     unsigned char* vc, int n_slots, int page) {
    using R = Q8Rows<T, D>;
    constexpr int kV = R::kV;
    __shared__ int sm_slot[1 + kQ8Most + kQ8Block], sm_run[kQ8Most], sm_count;   // a run: its first token, and 64 times its length
    const int t0 = blockIdx.x * tokens_per_cta, n = min(tokens_per_cta, n_tok - t0), tid = threadIdx.x, lane = tid & 31;
    grid_let_next_start();
    grid_wait_for_previous();
    if (tid == 0) sm_count = 0;
    if (tid < 1 + n + kQ8Block - 1) {
        const int t = t0 - 1 + tid, slot = t >= 0 && t < n_tok ? slots[t] : -1;
        sm_slot[tid] = slot < n_slots ? slot : -1;
    }
    __syncthreads();
    if (tid < n) {
        const int block = sm_slot[1 + tid] >> 4;   // (negative ones stay so)
        if (block >= 0 && sm_slot[tid] >> 4 != block) {
            int len = 1;
            while (len < kQ8Block && sm_slot[1 + tid + len] >> 4 == block) ++len;
            sm_run[atomicAdd(&sm_count, 1)] = tid | len << 6;
        }
    }
    __syncthreads();
    const bool second = blockIdx.y != 0;   // V
    const T* x = second ? v : k;
    const long long tok = second ? v_tok : k_tok, head = second ? v_head : k_head, page_bytes = q8_page_bytes(page, D);
    unsigned char* cache = second ? vc : kc;
    const int row = lane / R::kLanes, col = lane % R::kLanes * kV, units = sm_count * hkv;
    for (int unit = tid >> 5; unit < units; unit += kQ8Threads / 32) {
        const int i = unit / hkv, h = unit - i * hkv, first = sm_run[i] & 63, len = sm_run[i] >> 6;
        const int slot0 = sm_slot[1 + first], at_page = slot0 / page, in_page = (slot0 - at_page * page) & ~(kQ8Block - 1);
        unsigned char *begin = cache + ((long long)at_page * hkv + h) * page_bytes, *codes = begin + (long long)in_page * D, *power = begin + (long long)page * D + in_page / kQ8Block;
        const int was_byte = *power;
        // the run's values, and the largest finite one
        Q8Values<T> y[R::kLoads];
        unsigned top = 0;
        const T* from = x + (t0 + first + row) * tok + h * head + col;
#pragma unroll
        for (int j = 0; j < R::kLoads; ++j, from += R::kRows * tok) y[j].template load<kWide>(from, j * R::kRows + row < len);
#pragma unroll
        for (int j = 0; j < R::kLoads; ++j) top = y[j].largest(top);
        top = __reduce_max_sync(0xffffffffu, Q8Values<T>::bits(top));
        if (top >= 0x7f800000u) {   // infinities or NaN among them
            top = 0;
#pragma unroll
            for (int j = 0; j < R::kLoads; ++j)
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    const unsigned bits = __float_as_uint(y[j].get(e)) & 0x7fffffffu;
                    if (bits < 0x7f800000u) top = max(top, bits);
                }
            top = __reduce_max_sync(0xffffffffu, top);
        }
        const int mine = lane < len ? sm_slot[1 + first + lane] & (kQ8Block - 1) : -1;   // a token's row of the block
        const unsigned rows = __reduce_or_sync(0xffffffffu, mine >= 0 ? 1u << mine : 0u);
        const bool fresh = rows & 1;
        const int was = fresh ? kQ8Low : q8_exponent(was_byte), e = max(was, q8_exponent_of(top));
        if (!fresh && e > was) {   // the block's other rows, 16 bytes a lane
            const float by = q8_power(was - e);
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const int at = (j * 32 + lane) * 16;
                if (rows >> (at / D) & 1) continue;
                uint4 z = *reinterpret_cast<const uint4*>(codes + at);
                uint32_t w[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    float f[4];
                    q8_floats(w[m], f);
                    w[m] = q8_encode4(f[0] * by, f[1] * by, f[2] * by, f[3] * by);
                }
                *reinterpret_cast<uint4*>(codes + at) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        const float by = q8_power(-e);
#pragma unroll
        for (int j = 0; j < R::kLoads; ++j) {
            const int r = j * R::kRows + row;
            if (r < len) {
                uint32_t out[kV / 4];
#pragma unroll
                for (int m = 0; m < kV / 4; ++m)
                    out[m] = q8_encode4(y[j].get(4 * m) * by, y[j].get(4 * m + 1) * by, y[j].get(4 * m + 2) * by, y[j].get(4 * m + 3) * by);
                unsigned char* to = codes + (sm_slot[1 + first + r] & (kQ8Block - 1)) * D + col;
                if (kV == 8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[kV / 4 - 1]);
                else *reinterpret_cast<uint32_t*>(to) = out[0];
            }
        }
        __syncwarp();   // (every lane has read the byte)
        if (lane == 0 && (fresh || e + kQ8Bias != was_byte)) *power = (unsigned char)(e + kQ8Bias);
    }
}

// Where a token's rows are: those of head 0 of its page, and its row in the page; or one of
constexpr long long kQ8None = -1, kQ8Skip = -2;
struct Q8Place {
    long long begin;
    int row;
};
// kSectors: k and v start on 32 bytes
template <int D, bool kSectors>
__global__ void __launch_bounds__(kQ8Threads) cache_read_q8_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, const int* __restrict__ table,
                                                                   const int* __restrict__ cu, int B, int hkv, int n_pages, int page, int max_pages, int total,
                                                                   int tokens_per_cta, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v) {
    constexpr int kLanes = D / 16, kRows = kQ8Threads / kLanes, kAhead = 2;
    __shared__ Q8Place where[kQ8Threads];
    __shared__ int near[kQ8Threads];   // the counts of a small batch: a search step from memory takes as long as all of them
    const int t0 = blockIdx.x * tokens_per_cta, n = min(tokens_per_cta, total - t0), tid = threadIdx.x;
    const long long page_bytes = q8_page_bytes(page, D);
    grid_let_next_start();
    grid_wait_for_previous();
    const bool small = B < kQ8Threads;
    if (small && tid <= B) near[tid] = cu[tid];
    __syncthreads();
    if (tid < n) {
        const int t = t0 + tid;
        auto count = [&](int b) { return small ? near[b] : cu[b]; };
        Q8Place w{kQ8Skip, 0};
        if (t < count(B)) {
            int lo = 0, hi = B;   // the last b with cu[b] <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (count(mid) <= t) lo = mid;
                else hi = mid;
            }
            const int pos = t - count(lo), col = pos / page;
            const int p = pos >= 0 && col < max_pages ? table[(long long)lo * max_pages + col] : -1;
            w = Q8Place{p >= 0 && p < n_pages ? p * (hkv * page_bytes) : kQ8None, pos - col * page};
        }
        where[tid] = w;
    }
    __syncthreads();
    const int c = tid % kLanes, dt = kRows / hkv, dh = kRows - dt * hkv;
    long long to = ((long long)t0 * hkv + tid / kLanes) * D + c * 16;
    int t = tid / kLanes / hkv, h = tid / kLanes - t * hkv;
    while (t < n) {   // kAhead rows' loads, then their values
        uint4 x[kAhead][2];
        int powers[kAhead][2];
        unsigned there = 0;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
            powers[i][0] = powers[i][1] = 0;
            const Q8Place w = t < n ? where[t] : Q8Place{kQ8Skip, 0};
            if (w.begin != kQ8Skip) there |= 1u << i;
            if (w.begin >= 0) {
                const long long begin = w.begin + h * page_bytes, word = begin + (long long)w.row * D + c * 16, power = begin + (long long)page * D + w.row / kQ8Block;
                x[i][0] = *reinterpret_cast<const uint4*>(kc + word);
                x[i][1] = *reinterpret_cast<const uint4*>(vc + word);
                powers[i][0] = kc[power];
                powers[i][1] = vc[power];
            }
            t += dt;
            h += dh;
            if (h >= hkv) {
                h -= hkv;
                ++t;
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i, to += (long long)kRows * D) {
            if (!(there >> i & 1)) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float by = q8_power(q8_exponent(powers[i][j]));
                const uint32_t in[4] = {x[i][j].x, x[i][j].y, x[i][j].z, x[i][j].w};
                uint32_t out[8];
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    float f[4];
                    q8_floats(in[m], f);
                    out[2 * m] = sm100::pack_bf16x2(f[0] * by, f[1] * by);
                    out[2 * m + 1] = sm100::pack_bf16x2(f[2] * by, f[3] * by);
                }
                __nv_bfloat16* p = (j ? v : k) + to;
                if (kSectors) {
                    sm100::st_global_32B(p, out);
                } else {
                    *reinterpret_cast<uint4*>(p) = make_uint4(out[0], out[1], out[2], out[3]);
                    *reinterpret_cast<uint4*>(p + 8) = make_uint4(out[4], out[5], out[6], out[7]);
                }
            }
        }
    }
}

template <typename T, int D>
static cudaError_t launch_append(const CacheQ8& c, const void* k, const void* v, const long long (&ks)[2], const long long (&vs)[2], const int* slots, int T_, cudaStream_t st) {
    constexpr int kV = 16 / sizeof(T);
    bool wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    for (const long long* s : {ks, vs}) wide = wide && (T_ == 1 || s[0] % kV == 0) && (c.hkv == 1 || s[1] % kV == 0);
    const int resident = 2 * sm_count(), one_wave = (T_ + resident - 1) / resident, per = one_wave < kQ8Most ? one_wave : kQ8Most;
    auto go = [&](auto kernel) {
        LaunchScope ls(K_CACHE_APPEND_Q8, st);
        return launch_overlapped(kernel, dim3((unsigned)((T_ + per - 1) / per), 2), kQ8Threads, 0, st, (const T*)k, (const T*)v, slots, T_, per, c.hkv, ks[0], ks[1], vs[0], vs[1],
                                 (unsigned char*)c.k, (unsigned char*)c.v, c.n_pages * c.page_size, c.page_size);
    };
    return wide ? go(cache_append_q8_kernel<T, D, true>) : go(cache_append_q8_kernel<T, D, false>);
}
cudaError_t cache_append_q8(const CacheQ8& c, const void* k, const void* v, const long long (&ks)[2], const long long (&vs)[2], int bf16, const int* slots, int T,
                            cudaStream_t st) {
    if (c.D == 128) return bf16 ? launch_append<__nv_bfloat16, 128>(c, k, v, ks, vs, slots, T, st) : launch_append<float, 128>(c, k, v, ks, vs, slots, T, st);
    return bf16 ? launch_append<__nv_bfloat16, 64>(c, k, v, ks, vs, slots, T, st) : launch_append<float, 64>(c, k, v, ks, vs, slots, T, st);
}
cudaError_t cache_read_q8(const CacheQ8& c, const int* block_table, const int* cu, int B, int max_pages, int total, void* k, void* v, cudaStream_t st) {
    const int resident = 4 * sm_count(), one_wave = (total + resident - 1) / resident;
    int per = 128 / c.hkv;
    if (per > one_wave || 3 * per >= 2 * one_wave) per = one_wave;
    if (per < 1) per = 1;
    if (per > kQ8Threads) per = kQ8Threads;
    LaunchScope ls(K_CACHE_READ_Q8, st);
    auto go = [&](auto kernel) {
        return launch_overlapped(kernel, (unsigned)((total + per - 1) / per), kQ8Threads, 0, st, (const unsigned char*)c.k, (const unsigned char*)c.v, block_table, cu, B, c.hkv, c.n_pages,
                                 c.page_size, max_pages, total, per, (__nv_bfloat16*)k, (__nv_bfloat16*)v);
    };
    const bool sectors = (((uintptr_t)k | (uintptr_t)v) & 31) == 0;
    if (c.D == 128) return sectors ? go(cache_read_q8_kernel<128, true>) : go(cache_read_q8_kernel<128, false>);
    return sectors ? go(cache_read_q8_kernel<64, true>) : go(cache_read_q8_kernel<64, false>);
}

}  // namespace ttk
