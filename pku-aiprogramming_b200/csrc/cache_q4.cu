// Writing new keys and values into the 4-bit cache, and reading sequences back as packed bf16.
//
// Both are bound by HBM: D = 128 in bf16 is 256 bytes a token and head, its codes are 68.  A thread has eight channels -- one
// 16-byte access of bf16, one 4-byte word of the cache -- so a warp's accesses are whole rows on either side, and a group's
// maximum is over four neighbouring lanes.
#include "cache_q4.cuh"

namespace ttk {

constexpr int kQ4Threads = 256;

template <typename T, bool kWide>
__device__ __forceinline__ void q4_load8(const T* p, float (&x)[8]) {
    if (!kWide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
    } else if (sizeof(T) == 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    } else {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
}

// Eight channels of a group that four lanes share -> their word and the group's code; whole warps.  The levels are added up as they are, four bits
// apart: each is 1.5 2^23's bits plus -8 .. 7, and what that comes to without the levels' own 8 is a constant.
template <typename T>
__device__ __forceinline__ uint32_t q4_encode8(const float (&x)[8], int* code) {
    unsigned top = 0;   // bits of |x|: ordered as the values, with NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (top > 0x7f800000u) {
        *code = kQ4NaN;
        return 0x88888888u;
    }
    float s8;
    *code = q4_code(__uint_as_float(top), &s8);
    const float s = 0.125f * s8, inv = *code ? q4_reciprocal(s) : 0.f;
    const bool over = __uint_as_float(top) > 7.5f * s;   // beyond the largest scale
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float y = over ? fminf(fmaxf(x[i], -7.5f * s), 7.5f * s) : x[i];
        w = (w << 4) + (sizeof(T) == 2 ? q4_level_bf16(y, inv) : q4_level_f32(y, s, inv));
    }
    return w - kQ4Bits * 0x11111111u + 0x88888888u;
}

template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(kQ4Threads) cache_append_q4_kernel(const T* __restrict__ k, const T* __restrict__ v, const int* __restrict__ slots, unsigned rows,
                                                                     int hkv, long long k_tok, long long k_head, long long v_tok, long long v_head,
                                                                     unsigned char* __restrict__ kc, unsigned char* __restrict__ vc, int n_slots, int page) {
    constexpr int kLanes = D / 8, kRows = kQ4Threads / kLanes;
    const unsigned row = blockIdx.x * (unsigned)kRows + threadIdx.x / kLanes, t = row / (unsigned)hkv, h = row - t * (unsigned)hkv;
    const int c = threadIdx.x % kLanes;
    grid_let_next_start();
    grid_wait_for_previous();
    const int slot = row < rows ? slots[t] : -1;
    const bool here = slot >= 0 && slot < n_slots;
    float x[8] = {}, y[8] = {};
    if (here) {
        q4_load8<T, kWide>(k + t * k_tok + h * k_head + c * 8, x);
        q4_load8<T, kWide>(v + t * v_tok + h * v_head + c * 8, y);
    }
    int ck, cv;
    const uint32_t wk = q4_encode8<T>(x, &ck), wv = q4_encode8<T>(y, &cv);
    if (!here) return;
    const int p = slot / page, r = slot - p * page;
    const long long at = ((long long)p * hkv + h) * ((long long)page * q4_row_bytes(D));
    const long long word = at + r * (D / 2) + c * 4, code = at + (long long)page * (D / 2) + r * (D / 32) + c / 4;
    *reinterpret_cast<uint32_t*>(kc + word) = wk;
    *reinterpret_cast<uint32_t*>(vc + word) = wv;
    if (c % 4 == 0) {
        kc[code] = (unsigned char)ck;
        vc[code] = (unsigned char)cv;
    }
}

template <int D>
__global__ void __launch_bounds__(kQ4Threads) cache_read_q4_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, const int* __restrict__ table,
                                                                   const int* __restrict__ cu, int B, int hkv, int n_pages, int page, int max_pages, int total,
                                                                   int tokens_per_cta, uint32_t k128, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v) {   // k128: 0x43004300, in a register
    constexpr int kLanes = D / 8, kRows = kQ4Threads / kLanes;
    __shared__ int2 where[kQ4Threads];   // of each token of the CTA its page and row in it; page -1: zeros, -2: left alone
    const int t0 = blockIdx.x * tokens_per_cta, n = min(tokens_per_cta, total - t0);
    grid_let_next_start();
    grid_wait_for_previous();
    if (threadIdx.x < n) {
        const int t = t0 + threadIdx.x;
        int2 w = make_int2(-2, 0);
        if (t < cu[B]) {
            int lo = 0, hi = B;   // the last b with cu[b] <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int pos = t - cu[lo], col = pos / page;
            const int p = pos >= 0 && col < max_pages ? table[(long long)lo * max_pages + col] : -1;
            w = make_int2(p >= 0 && p < n_pages ? p : -1, pos - col * page);
        }
        where[threadIdx.x] = w;
    }
    __syncthreads();
    const int c = threadIdx.x % kLanes;
    const unsigned rows = (unsigned)n * (unsigned)hkv;
    for (unsigned row = threadIdx.x / kLanes; row < rows; row += kRows) {
        const unsigned t = row / (unsigned)hkv, h = row - t * (unsigned)hkv;
        const int2 w = where[t];
        if (w.x == -2) continue;
        const long long to = ((long long)t0 * hkv + row) * D + c * 8;
        const long long at = ((long long)w.x * hkv + h) * ((long long)page * q4_row_bytes(D));
        const long long word = at + w.y * (D / 2) + c * 4, code = at + (long long)page * (D / 2) + w.y * (D / 32) + c / 4;
        uint32_t x[2] = {0x88888888u, 0x88888888u}, codes[2] = {0, 0};
        if (w.x >= 0) {
            x[0] = *reinterpret_cast<const uint32_t*>(kc + word);
            x[1] = *reinterpret_cast<const uint32_t*>(vc + word);
            codes[0] = kc[code];
            codes[1] = vc[code];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // 0x4300 | n is 128 + n in bf16; (128 + n) s - 136 s, exactly: 17 times four bits has eight
            const __nv_bfloat162 s = __float2bfloat162_rn(0.125f * q4_scale8((int)codes[i])), off = __hmul2(s, __float2bfloat162_rn(-136.f));
            uint32_t y[4];   // channels j and j + 4
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y[j]) : "r"(x[i] >> (4 * j)), "n"(0x000f000f), "r"(k128));
                const __nv_bfloat162 z = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&y[j]), s, off);
                y[j] = *reinterpret_cast<const uint32_t*>(&z);
            }
            const uint4 out = make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632));
            *reinterpret_cast<uint4*>((i ? v : k) + to) = out;
        }
    }
}

template <typename T, int D>
static cudaError_t launch_append(const CacheQ4& c, const void* k, const void* v, const long long (&ks)[2], const long long (&vs)[2], const int* slots, int T_,
                                 cudaStream_t st) {
    constexpr int kRows = kQ4Threads / (D / 8), kV = 16 / sizeof(T);
    const unsigned rows = (unsigned)T_ * (unsigned)c.hkv;
    bool wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    for (const long long* s : {ks, vs}) wide = wide && (T_ == 1 || s[0] % kV == 0) && (c.hkv == 1 || s[1] % kV == 0);
    auto go = [&](auto kernel) {
        LaunchScope ls(K_CACHE_APPEND, st);
        return launch_overlapped(kernel, (rows + kRows - 1) / kRows, kQ4Threads, 0, st, (const T*)k, (const T*)v, slots, rows, c.hkv, ks[0], ks[1], vs[0], vs[1],
                                 (unsigned char*)c.k, (unsigned char*)c.v, c.n_pages * c.page_size, c.page_size);
    };
    return wide ? go(cache_append_q4_kernel<T, D, true>) : go(cache_append_q4_kernel<T, D, false>);
}
cudaError_t cache_append_q4(const CacheQ4& c, const void* k, const void* v, const long long (&ks)[2], const long long (&vs)[2], int bf16, const int* slots, int T,
                            cudaStream_t st) {
    if (c.D == 128) return bf16 ? launch_append<__nv_bfloat16, 128>(c, k, v, ks, vs, slots, T, st) : launch_append<float, 128>(c, k, v, ks, vs, slots, T, st);
    return bf16 ? launch_append<__nv_bfloat16, 64>(c, k, v, ks, vs, slots, T, st) : launch_append<float, 64>(c, k, v, ks, vs, slots, T, st);
}
cudaError_t cache_read_q4(const CacheQ4& c, const int* block_table, const int* cu, int B, int max_pages, int total, void* k, void* v, cudaStream_t st) {
    // about 128 rows per CTA, so that its look-ups are few and its loads many; fewer where that leaves SMs without one
    int per = 128 / c.hkv, spread = (total + 4 * sm_count() - 1) / (4 * sm_count());
    if (per > spread) per = spread;
    if (per < 1) per = 1;
    const unsigned grid = (unsigned)((total + per - 1) / per);
    LaunchScope ls(K_CACHE_READ, st);
    auto go = [&](auto kernel) {
        return launch_overlapped(kernel, grid, kQ4Threads, 0, st, (const unsigned char*)c.k, (const unsigned char*)c.v, block_table, cu, B, c.hkv, c.n_pages, c.page_size,
                                 max_pages, total, per, 0x43004300u, (__nv_bfloat16*)k, (__nv_bfloat16*)v);
    };
    return c.D == 128 ? go(cache_read_q4_kernel<128>) : go(cache_read_q4_kernel<64>);
}

}  // namespace ttk
