// Writing new keys and values into the 4-bit cache, and reading sequences back as packed bf16.
//
// Both are bound by HBM -- D = 128 in bf16 is 256 bytes a token and head, its codes are 68 -- once the arithmetic is out of the way.  In writing
// that is the work per group, so a thread has a whole one (32 channels, K and V apart): 20,000 tokens of 8 heads 34.8 us with four lanes to a
// group, which meet for its maximum, 21.5 so, 19.8 with bf16 kept in pairs (40 registers for 64).  In reading it is the number of memory instructions: a whole group to a thread there too, as 16 bytes
// and one, and four stores of a sector each.
#include "cache_q4.cuh"
#include "sm100_ptx.cuh"

namespace ttk {

constexpr int kQ4Threads = 256;

// 32 channels of a group as they come, bf16 in pairs.
template <typename T> struct Q4Group;
template <> struct Q4Group<__nv_bfloat16> {
    uint32_t w[16];
    template <bool kWide> __device__ __forceinline__ void load(const __nv_bfloat16* p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (kWide) {
                const uint4 r = *reinterpret_cast<const uint4*>(p + 8 * i);
                w[4 * i] = r.x; w[4 * i + 1] = r.y; w[4 * i + 2] = r.z; w[4 * i + 3] = r.w;
            } else {
                const unsigned short* q = reinterpret_cast<const unsigned short*>(p) + 8 * i;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = q[2 * j] | (uint32_t)q[2 * j + 1] << 16;
            }
        }
    }
    __device__ __forceinline__ void chunk(int i, uint4 r) { w[4 * i] = r.x; w[4 * i + 1] = r.y; w[4 * i + 2] = r.z; w[4 * i + 3] = r.w; }
    __device__ __forceinline__ unsigned top() const {   // the bits of the largest |x|: ordered as the values, with NaN above infinity
        uint32_t y = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) y = __vmaxu2(y, w[i] & 0x7fff7fffu);
        return max(y << 16, y & 0xffff0000u);
    }
    __device__ __forceinline__ float get(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
    __device__ __forceinline__ void put(int i, float x) {   // x exact in bf16
        const uint32_t y = __float_as_uint(x);
        w[i >> 1] = i & 1 ? (w[i >> 1] & 0xffffu) | y : (w[i >> 1] & 0xffff0000u) | y >> 16;
    }
};
template <> struct Q4Group<float> {
    float x[32];
    template <bool kWide> __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (kWide) {
                const float4 r = *reinterpret_cast<const float4*>(p + 4 * i);
                x[4 * i] = r.x; x[4 * i + 1] = r.y; x[4 * i + 2] = r.z; x[4 * i + 3] = r.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * i + j] = p[4 * i + j];
            }
        }
    }
    __device__ __forceinline__ void chunk(int i, uint4 r) {
        x[4 * i] = __uint_as_float(r.x); x[4 * i + 1] = __uint_as_float(r.y); x[4 * i + 2] = __uint_as_float(r.z); x[4 * i + 3] = __uint_as_float(r.w);
    }
    __device__ __forceinline__ unsigned top() const {
        unsigned y = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) y = max(y, __float_as_uint(x[i]) & 0x7fffffffu);
        return y;
    }
    __device__ __forceinline__ float get(int i) const { return x[i]; }
    __device__ __forceinline__ void put(int i, float y) { x[i] = y; }
};

// A group's four words and its code.  The levels are added up as they are, four bits apart: each is 1.5 2^23's bits plus -8 .. 7, and what that comes
// to without the levels' own 8 is a constant.
template <typename T>
__device__ __forceinline__ uint4 q4_encode(Q4Group<T>& x, int* code) {
    const unsigned top = x.top();
    float s8;
    *code = q4_code(__uint_as_float(min(top, 0x7f800000u)), &s8);
    const float s = 0.125f * s8, inv = !*code ? 0.f : sizeof(T) == 2 ? q4_reciprocal(s) : __frcp_rn(s);
    if (!(__uint_as_float(top) <= 7.5f * s)) {   // beyond the largest scale (7.5 of which, 6720, bf16 holds), or no number
        if (top > 0x7f800000u) *code = kQ4NaN;
#pragma unroll
        for (int i = 0; i < 32; ++i) x.put(i, top > 0x7f800000u ? 0.f : fminf(fmaxf(x.get(i), -7.5f * s), 7.5f * s));
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[j] = 0;
#pragma unroll
        for (int i = 7; i >= 0; --i) w[j] = (w[j] << 4) + (sizeof(T) == 2 ? q4_level_bf16(x.get(8 * j + i), inv) : q4_level_f32(x.get(8 * j + i), s, inv));
        w[j] += 0x88888888u - kQ4Bits * 0x11111111u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Where a token's rows are: those of head 0 of its page, and its row in the page; or one of
constexpr long long kQ4None = -1, kQ4Skip = -2;
struct Q4Place {
    long long begin;
    int row;
};
// A thread's walk over (token, head) rows, kRows apart.
struct Q4Walk {
    int t, h, dt, dh, hkv;
    __device__ __forceinline__ Q4Walk(int row, int rows_apart, int heads) : t(row / heads), dt(rows_apart / heads), hkv(heads) {
        h = row - t * heads;
        dh = rows_apart - dt * heads;
    }
    __device__ __forceinline__ void next() {
        t += dt;
        h += dh;
        if (h >= hkv) {
            h -= hkv;
            ++t;
        }
    }
};

// (Four CTAs per SM with floats: 36.0 us for 38.9 at 20,000 tokens of 8 heads of 128, where the compiler would take 79 registers.)
template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(kQ4Threads, kWide && sizeof(T) == 4 ? 4 : 0) cache_append_q4_kernel(const T* __restrict__ k, const T* __restrict__ v, const int* __restrict__ slots, int n_tok, int tokens_per_cta,
                                                                     int hkv, long long k_tok, long long k_head, long long v_tok, long long v_head,
                                                                     unsigned char* __restrict__ kc, unsigned char* __restrict__ vc, int n_slots, int page) {
    constexpr int kLanes = D / 32, kRows = kQ4Threads / kLanes, kChunks = 2 * sizeof(T);   // 16 bytes each, of a group
    // A group of floats is a whole line of 128 bytes, so a load of 16 bytes by a thread for itself would touch as many lines as lanes: the lanes of a row
    // load it together and exchange through shared memory, chunks moved about by the group so that both ways are without bank conflicts (a line has two
    // groups of bf16, where this costs more than it gives: 22.5 us for 19.9).
    constexpr bool kStaged = kWide && sizeof(T) == 4;
    __shared__ Q4Place where[kQ4Threads];
    __shared__ uint4 stage[kStaged ? kRows : 1][kLanes * kChunks + kLanes];
    const int t0 = blockIdx.x * tokens_per_cta, n = min(tokens_per_cta, n_tok - t0), c = threadIdx.x % kLanes;
    uint4* staged = stage[kStaged ? threadIdx.x / kLanes : 0];
    const unsigned row_lanes = ((1u << kLanes) - 1) << (threadIdx.x % 32 / kLanes * kLanes);
    const long long page_bytes = (long long)page * q4_row_bytes(D);
    const bool second = blockIdx.y != 0;   // V
    const T* from = (second ? v : k) + t0 * (second ? v_tok : k_tok) + (kStaged ? 0 : c * 32);
    const long long tok = second ? v_tok : k_tok, head = second ? v_head : k_head;
    unsigned char* into = second ? vc : kc;
    grid_let_next_start();
    grid_wait_for_previous();
    if (threadIdx.x < n) {
        const int slot = slots[t0 + threadIdx.x], p = slot / page;
        where[threadIdx.x] = Q4Place{slot >= 0 && slot < n_slots ? p * (hkv * page_bytes) : kQ4Skip, slot - p * page};
    }
    __syncthreads();
    for (Q4Walk at(threadIdx.x / kLanes, kRows, hkv); at.t < n; at.next()) {
        const Q4Place w = where[at.t];
        if (w.begin == kQ4Skip) continue;
        Q4Group<T> x;
        if constexpr (kStaged) {
            uint4 y[kChunks];
            const uint4* p = reinterpret_cast<const uint4*>(from + at.t * tok + at.h * head);
#pragma unroll
            for (int i = 0; i < kChunks; ++i) y[i] = p[i * kLanes + c];
            __syncwarp(row_lanes);   // (the row before has been read)
#pragma unroll
            for (int i = 0; i < kChunks; ++i) staged[(i * kLanes + c) ^ ((i * kLanes + c) / kChunks)] = y[i];
            __syncwarp(row_lanes);
#pragma unroll
            for (int i = 0; i < kChunks; ++i) x.chunk(i, staged[(c * kChunks + i) ^ c]);
        } else {
            x.template load<kWide>(from + at.t * tok + at.h * head);
        }
        int code;
        const uint4 words = q4_encode<T>(x, &code);
        unsigned char* to = into + w.begin + at.h * page_bytes;
        *reinterpret_cast<uint4*>(to + w.row * (D / 2) + c * 16) = words;
        to[(long long)page * (D / 2) + w.row * (D / 32) + c] = (unsigned char)code;
    }
}

// kSectors: k and v start on 32 bytes
template <int D, bool kSectors>
__global__ void __launch_bounds__(kQ4Threads) cache_read_q4_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, const int* __restrict__ table,
                                                                   const int* __restrict__ cu, int B, int hkv, int n_pages, int page, int max_pages, int total,
                                                                   int tokens_per_cta, uint32_t k128, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v) {   // k128: 0x43004300, in a register
    constexpr int kLanes = D / 32, kRows = kQ4Threads / kLanes, kAhead = 2;
    __shared__ Q4Place where[kQ4Threads];
    __shared__ int near[kQ4Threads];   // the counts of a small batch: a search step from memory takes as long as all of them
    const int t0 = blockIdx.x * tokens_per_cta, n = min(tokens_per_cta, total - t0);
    const long long page_bytes = (long long)page * q4_row_bytes(D);
    grid_let_next_start();
    grid_wait_for_previous();
    const bool small = B < kQ4Threads;
    if (small && threadIdx.x <= B) near[threadIdx.x] = cu[threadIdx.x];
    __syncthreads();
    if (threadIdx.x < n) {
        const int t = t0 + threadIdx.x;
        auto count = [&](int b) { return small ? near[b] : cu[b]; };
        Q4Place w{kQ4Skip, 0};
        if (t < count(B)) {
            int lo = 0, hi = B;   // the last b with cu[b] <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (count(mid) <= t) lo = mid;
                else hi = mid;
            }
            const int pos = t - count(lo), col = pos / page;
            const int p = pos >= 0 && col < max_pages ? table[(long long)lo * max_pages + col] : -1;
            w = Q4Place{p >= 0 && p < n_pages ? p * (hkv * page_bytes) : kQ4None, pos - col * page};
        }
        where[threadIdx.x] = w;
    }
    __syncthreads();
    const int c = threadIdx.x % kLanes;
    long long to = ((long long)t0 * hkv + threadIdx.x / kLanes) * D + c * 32;
    Q4Walk at(threadIdx.x / kLanes, kRows, hkv);
    while (at.t < n) {   // kAhead rows' loads, then their values
        uint4 x[kAhead][2];
        uint32_t codes[kAhead][2];
        unsigned there = 0;
#pragma unroll
        for (int i = 0; i < kAhead; ++i, at.next()) {
            x[i][0] = x[i][1] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
            codes[i][0] = codes[i][1] = 0;
            const Q4Place w = at.t < n ? where[at.t] : Q4Place{kQ4Skip, 0};
            if (w.begin != kQ4Skip) there |= 1u << i;
            if (w.begin >= 0) {
                const long long begin = w.begin + at.h * page_bytes, word = begin + w.row * (D / 2) + c * 16, code = begin + (long long)page * (D / 2) + w.row * (D / 32) + c;
                x[i][0] = *reinterpret_cast<const uint4*>(kc + word);
                x[i][1] = *reinterpret_cast<const uint4*>(vc + word);
                codes[i][0] = kc[code];
                codes[i][1] = vc[code];
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i, to += kRows * D) {
            if (!(there >> i & 1)) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // 0x4300 | n is 128 + n in bf16; (128 + n) s - 136 s, exactly: 17 times four bits has eight
                const __nv_bfloat162 s = __float2bfloat162_rn(0.125f * q4_scale8((int)codes[i][j])), off = __hmul2(s, __float2bfloat162_rn(-136.f));
                const uint32_t in[4] = {x[i][j].x, x[i][j].y, x[i][j].z, x[i][j].w};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t out[8];
#pragma unroll
                    for (int word = 0; word < 2; ++word) {
                        uint32_t y[4];   // channels m and m + 4
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y[m]) : "r"(in[2 * half + word] >> (4 * m)), "n"(0x000f000f), "r"(k128));
                            const __nv_bfloat162 z = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&y[m]), s, off);
                            y[m] = *reinterpret_cast<const uint32_t*>(&z);
                        }
                        out[4 * word] = __byte_perm(y[0], y[1], 0x5410);
                        out[4 * word + 1] = __byte_perm(y[2], y[3], 0x5410);
                        out[4 * word + 2] = __byte_perm(y[0], y[1], 0x7632);
                        out[4 * word + 3] = __byte_perm(y[2], y[3], 0x7632);
                    }
                    __nv_bfloat16* p = (j ? v : k) + to + 16 * half;
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
}

// Tokens per CTA: about 128 rows, so that look-ups are few beside them; fewer where all CTAs are resident at once then (`resident` of them), and more, up
// to half as many again, where that leaves no second wave.  20,000 tokens of 8 heads, D = 128: writing bf16 20.8 / 19.8 / 21.9 / 22.8 us at 64 / 128 /
// 256 / 512 rows (5.3 TB/s at 128), float 35.7 at 128 (46.1 with every lane's loads its own; 5.2 TB/s); 47,000 tokens: reading 39.5 / 43.6 / 46.3 at 128 /
// 256 / 512 (6.0 TB/s at 128).  One wave, for what 128 rows and four CTAs per SM take: writing 8628 tokens of one head 3.2 for 4.4, 6801 of four 4.9 for
// 5.7, 1000 of two of 64 floats 2.2 for 3.8; reading 25,070 of four heads 12.1 for 13.8.
static int q4_tokens_per_cta(int tokens, int hkv, int resident) {
    int per = 128 / hkv;
    const int one_wave = (tokens + resident - 1) / resident;
    if (per > one_wave || 3 * per >= 2 * one_wave) per = one_wave;
    return per < 1 ? 1 : per;
}

template <typename T, int D>
static cudaError_t launch_append(const CacheQ4& c, const void* k, const void* v, const long long (&ks)[2], const long long (&vs)[2], const int* slots, int T_,
                                 cudaStream_t st) {
    constexpr int kV = 16 / sizeof(T);
    bool wide = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    for (const long long* s : {ks, vs}) wide = wide && (T_ == 1 || s[0] % kV == 0) && (c.hkv == 1 || s[1] % kV == 0);
    const int per = q4_tokens_per_cta(T_, c.hkv, (wide && sizeof(T) == 2 ? 6 : wide ? 4 : 3) * sm_count() / 2);
    auto go = [&](auto kernel) {
        LaunchScope ls(K_CACHE_APPEND, st);
        return launch_overlapped(kernel, dim3((unsigned)((T_ + per - 1) / per), 2), kQ4Threads, 0, st, (const T*)k, (const T*)v, slots, T_, per, c.hkv, ks[0], ks[1], vs[0], vs[1],
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
    const int per = q4_tokens_per_cta(total, c.hkv, 5 * sm_count());
    const unsigned grid = (unsigned)((total + per - 1) / per);
    LaunchScope ls(K_CACHE_READ, st);
    auto go = [&](auto kernel) {
        return launch_overlapped(kernel, grid, kQ4Threads, 0, st, (const unsigned char*)c.k, (const unsigned char*)c.v, block_table, cu, B, c.hkv, c.n_pages, c.page_size,
                                 max_pages, total, per, 0x43004300u, (__nv_bfloat16*)k, (__nv_bfloat16*)v);
    };
    const bool sectors = (((uintptr_t)k | (uintptr_t)v) & 31) == 0;
    if (c.D == 128) return sectors ? go(cache_read_q4_kernel<128, true>) : go(cache_read_q4_kernel<128, false>);
    return sectors ? go(cache_read_q4_kernel<64, true>) : go(cache_read_q4_kernel<64, false>);
}

}  // namespace ttk
