// Single-query attention over the 4-bit key/value cache: out = softmax(scale q K^T) V with K, V = (n - 8) s.
//
// A key and key/value head are 2 (D / 2 + D / 32) bytes, at D = 128 136 of them for 256 values.  At the measured copy rate an SM
// gets 23 bytes a cycle, so it has 5.9 cycles for those 256 values: what bounds this next to HBM is the instructions that turn
// nibbles into operands.  So nothing else is done to them: a lane loads exactly the nibbles that are its elements of the
// tensor-core operand (mma.sync m16n8k16: the accumulators are 16 x 8, so up to eight query heads of a group fill it;
// operands that are made in registers would have to go through shared memory or tensor memory for tcgen05, 512 more bytes a
// key), and the order of channels within a product is chosen so that they are one 16-byte load of one scale.
//
//   S^T [16 keys x 8 heads] += K [16 keys x 16 channels] Q^T: lane (g, t) of a warp (g = lane / 4, t = lane % 4) holds of keys g and
//     g + 8 the quarter t of the channels; k-step j takes two words' pairs (channels i and i + 4 of eight).
//   O^T [16 channels x 8 heads] += V^T [16 channels x 16 keys] P^T: lane (g, t) holds of keys 2t, 2t + 1, 2t + 8, 2t + 9 the eighth g of the
//     channels, and so its part of the result is D / 8 neighbouring channels of heads 2t and 2t + 1.
//
// Nibbles become halves by their bits: 0x6400 | n is 1024 + n, 0x6400 | n << 4 is 1024 + 16 n, so one logical instruction makes two
// halves, and one or two half operations make (n - 8) s of them, exactly: s has four significant bits, n - 8 four.  q's exponent is
// moved so that every bf16 value of a head that matters is exact in half.  Softmax is online in base 2; the reference is raised, for
// all of a warp's heads, when a score passes it by 2^kSlack, and P is taken 2^kLift higher, up to 2^15: rounded to half it is off
// by 2^-11 of itself (bf16: 2^-8) down to 2^-24 of the row's largest, and by 2^-35 of that below.  Accumulators are 32-bit.
//
// A warp takes every fourth 32 keys of its CTA's range; four warps and then the ranges are merged.
#include "cache_q4.cuh"
#include "sm100_ptx.cuh"

namespace ttk {
using namespace sm100;

namespace {

constexpr int kWarps = 4, kTile = 32;   // keys per warp and step: two accumulator tiles of 16
constexpr float kSlack = 5.f, kLift = 10.f;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ half2 as_half2(uint32_t x) { return *reinterpret_cast<half2*>(&x); }
__device__ __forceinline__ uint32_t bits(half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// A word's eight nibbles, the i-th of the low half beside the i-th of the high half, times the scales of the two halves: `s8` holds
// half(code << 7), eight times them.  The codes that are written (and NaN) leave every constant finite: 9 s8 <= 64512.
struct Scale2 {
    half2 s8, a, b;
    __device__ __forceinline__ explicit Scale2(uint32_t codes_times_128) {
        s8 = as_half2(codes_times_128);
        a = __hmul2(s8, __float2half2_rn(1.f / 128));
        b = __hmul2(s8, __float2half2_rn(-9.f));
    }
};
__device__ __forceinline__ void unpack_q4(uint32_t x, const Scale2& s, uint32_t (&out)[4]) {
    const uint32_t y = x >> 8;
    const half2 eighth = __float2half2_rn(0.125f), off = __float2half2_rn(-129.f);
    // (1024 + n) / 8 - 129 = (n - 8) / 8;  (1024 + 16 n) s8 / 128 - 9 s8 = (n - 8) s8 / 8
    out[0] = bits(__hmul2(__hfma2(as_half2((x & 0x000f000fu) | 0x64006400u), eighth, off), s.s8));
    out[1] = bits(__hfma2(as_half2((x & 0x00f000f0u) | 0x64006400u), s.a, s.b));
    out[2] = bits(__hmul2(__hfma2(as_half2((y & 0x000f000fu) | 0x64006400u), eighth, off), s.s8));
    out[3] = bits(__hfma2(as_half2((y & 0x00f000f0u) | 0x64006400u), s.a, s.b));
}

// The bytes of 16 keys that a lane needs, as loaded.
template <int D>
struct Raw16 {
    static constexpr int kKW = D / 32, kVW = D / 64;   // words per key of a lane
    uint32_t k[2][kKW], v[4][kVW];
    uint32_t kc[2];          // codes of the lane's quarter of keys g, g + 8
    uint32_t vc[2][D / 64];  // codes of keys 2t, 2t + 1 and of 2t + 8, 2t + 9
};
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char* p) {
    if (N == 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = x.x; w[1 % N] = x.y; w[2 % N] = x.z; w[3 % N] = x.w;
    } else if (N == 2) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = x.x; w[1 % N] = x.y;
    } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
}

}  // namespace

struct DecodeQ4Args {
    const __nv_bfloat16* q;
    const unsigned char *kc, *vc;
    const int *table, *lens;
    int L, hkv, group, head_tiles, n_pages, page, max_pages, splits, chunk;
    float scale_log2;
    __nv_bfloat16* out;   // splits == 1
    float* lse;           // may be null then
    float *po, *plse;     // splits > 1: normalised rows [slice, split, group, D] and log-sum-exps
};

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32) attn_decode_q4_kernel(const DecodeQ4Args a) {
    constexpr int kHeads = 8 * NT, kKW = D / 32, kVW = D / 64, kMT = D / 16;
    __shared__ float sm_o[kWarps][kHeads][D + 4];
    __shared__ float sm_m[kWarps][kHeads], sm_l[kWarps][kHeads];
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp_idx(), g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % a.splits, item = blockIdx.x / a.splits, tile = item % a.head_tiles, slice = item / a.head_tiles;
    const int b = slice / a.hkv, hk = slice - b * a.hkv, h0 = tile * kHeads, n_heads = min(kHeads, a.group - h0);
    grid_let_next_start();
    grid_wait_for_previous();
    const int len = a.lens ? min(max(a.lens[b], 0), a.L) : a.L;
    const int k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
    const long long row0 = (long long)slice * a.group + h0;   // the tile's first query head

    // query heads as the B operand: lane (g, t) has head g's quarter t of the channels, pairs (i, i + 4) of eight
    uint32_t qf[NT][kKW][4];
    float to_log2[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        uint4 w[kKW];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kKW; ++i) {
            w[i] = g + 8 * n < n_heads ? __ldg(reinterpret_cast<const uint4*>(a.q + (row0 + g + 8 * n) * D + t * (D / 4)) + i) : make_uint4(0, 0, 0, 0);
            const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x[j] << 16)), fabsf(__uint_as_float(x[j] & 0xffff0000u))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the head's largest value to 2^14 .. 2^15 (zeros and infinities as they are)
        const int e = (int)(__float_as_uint(top) >> 23) - 127, up = top > 0.f && e < 128 ? min(max(14 - e, -100), 100) : 0;
        const float f = __uint_as_float((unsigned)(up + 127) << 23), back = __uint_as_float((unsigned)(127 - up) << 23);
#pragma unroll
        for (int i = 0; i < kKW; ++i) {
            auto pair = [&](uint32_t lo, uint32_t hi, bool upper) {
                const float x = upper ? __uint_as_float(lo & 0xffff0000u) : __uint_as_float(lo << 16), y = upper ? __uint_as_float(hi & 0xffff0000u) : __uint_as_float(hi << 16);
                return bits(__floats2half2_rn(x * f, y * f));
            };
            qf[n][i][0] = pair(w[i].x, w[i].z, false);
            qf[n][i][1] = pair(w[i].x, w[i].z, true);
            qf[n][i][2] = pair(w[i].y, w[i].w, false);
            qf[n][i][3] = pair(w[i].y, w[i].w, true);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) to_log2[n][j] = a.scale_log2 * __shfl_sync(0xffffffffu, back, (2 * t + j) * 4);
    }

    float o[kMT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][n][j] = 0.f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
    }

    // 16 keys lie in one page.  Lane i looks up the page of the i-th 16 keys from `batch` on; the page -1 has no keys.
    const int n_sub = k1 > k0 ? ((k1 - k0 + kTile - 1) / kTile + kWarps - 1 - warp) / kWarps * 2 : 0;   // this warp's 16-key tiles
    auto first_key = [&](int sub) { return k0 + ((sub >> 1) * kWarps + warp) * kTile + (sub & 1) * 16; };
    auto look_up = [&](int sub, int& page, int& row) {
        const int key = first_key(sub);
        page = -1;
        row = 0;
        if (sub < n_sub && key < k1) {
            const int col = key / a.page;
            row = key - col * a.page;
            if (a.table) page = col < a.max_pages ? __ldg(a.table + (long long)b * a.max_pages + col) : -1;
            else page = b;
            if (page >= a.n_pages) page = -1;
        }
    };
    const long long page_bytes = (long long)a.page * q4_row_bytes(D);
    const int codes_at = a.page * (D / 2);
    auto load = [&](int page, int row, Raw16<D>& r) {
        if (page < 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                r.kc[i] = 0;
#pragma unroll
                for (int j = 0; j < kKW; ++j) r.k[i][j] = 0;
#pragma unroll
                for (int j = 0; j < D / 64; ++j) r.vc[i][j] = 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kVW; ++j) r.v[i][j] = 0;
            return;
        }
        const long long at = ((long long)page * a.hkv + hk) * page_bytes;
        const unsigned char *kp = a.kc + at, *vp = a.vc + at;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            load_words<kKW>(r.k[i], kp + (row + g + 8 * i) * (D / 2) + t * (D / 8));
            r.kc[i] = __ldg(kp + codes_at + (row + g + 8 * i) * (D / 32) + t * (D / 32) / 4);
            load_words<D / 64>(r.vc[i], vp + codes_at + (row + 2 * t + 8 * i) * (D / 32));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<kVW>(r.v[i], vp + (row + 2 * t + (i & 1) + (i >> 1) * 8) * (D / 2) + g * (D / 16));
    };

    int page_now, row_now;   // of the batch that holds the tile being loaded
    look_up(lane, page_now, row_now);
    auto fetch = [&](int sub, Raw16<D>& r) -> bool {
        const int page = __shfl_sync(0xffffffffu, page_now, sub & 31), row = __shfl_sync(0xffffffffu, row_now, sub & 31);
        load(page, row, r);
        return page >= 0;
    };
    Raw16<D> next[2];
    bool there[2] = {false, false};
    if (n_sub > 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) there[i] = fetch(i, next[i]);
    }

    for (int sub = 0; sub < n_sub; sub += 2) {
        Raw16<D> raw[2] = {next[0], next[1]};
        const bool here[2] = {there[0], there[1]};
        if (sub + 2 < n_sub) {
            if (((sub + 2) & 31) == 0) look_up(sub + 2 + lane, page_now, row_now);
#pragma unroll
            for (int i = 0; i < 2; ++i) there[i] = fetch(sub + 2 + i, next[i]);
        }
        // scores
        float s[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[u][n][j] = 0.f;
            const Scale2 lo(raw[u].kc[0] * 0x00800080u), hi(raw[u].kc[1] * 0x00800080u);
#pragma unroll
            for (int w = 0; w < kKW; ++w) {
                uint32_t x[4], y[4];
                unpack_q4(raw[u].k[0][w], lo, x);
                unpack_q4(raw[u].k[1][w], hi, y);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16816(s[u][n], x[0], y[0], x[1], y[1], qf[n][w][0], qf[n][w][1]);
                    mma16816(s[u][n], x[2], y[2], x[3], y[3], qf[n][w][2], qf[n][w][3]);
                }
            }
        }
        // keys behind the range, or without a page: no score, and scales of 0 so that what lies there does not meet P = 0
        if (first_key(sub) + kTile > k1 || !here[0] || !here[1]) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int left = here[u] ? k1 - first_key(sub + u) : 0;   // keys of these 16
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (g + (j >> 1) * 8 >= left) s[u][n][j] = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = 2 * t + 8 * i;
                    if (D == 128) {
                        if (key >= left) raw[u].vc[i][0] = 0;
                        if (key + 1 >= left) raw[u].vc[i][D / 64 - 1] = 0;
                    } else {
                        if (key >= left) raw[u].vc[i][0] = 0;
                        else if (key + 1 >= left) raw[u].vc[i][0] &= 0xffffu;
                    }
                }
            }
        }
        // the maximum, where a score passes it by 2^8
        bool raise = false;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[n][j] = fmaxf(fmaxf(s[0][n][j], s[0][n][j + 2]), fmaxf(s[1][n][j], s[1][n][j + 2])) * to_log2[n][j];
                raise = raise || top[n][j] > m[n][j] + kSlack;
            }
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = top[n][j];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    const float to = fmaxf(m[n][j], x), f = m[n][j] == to ? 1.f : ex2_approx(m[n][j] - to);
                    m[n][j] = to;
                    l[n][j] *= f;
#pragma unroll
                    for (int i = 0; i < kMT; ++i) {
                        o[i][n][j] *= f;
                        o[i][n][j + 2] *= f;
                    }
                }
            }
        }
        // P^T as the B operand
        uint32_t p[2][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0] - kLift, m1 = m[n][1] == -INFINITY ? 0.f : m[n][1] - kLift;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = ex2_approx(fmaf(s[u][n][2 * i], to_log2[n][0], -m0)), y = ex2_approx(fmaf(s[u][n][2 * i + 1], to_log2[n][1], -m1));
                    l[n][0] += x;
                    l[n][1] += y;
                    p[u][n][i] = transposed8x8(bits(__floats2half2_rn(x, y)));
                }
            }
        }
        // O^T
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // the two keys' codes of the lane's group of channels, times 128, in the two halves of a word
            uint32_t c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (D == 128) c[i] = __byte_perm(raw[u].vc[i][0], raw[u].vc[i][D / 64 - 1], (g >> 1) | (4 + (g >> 1)) << 8);
                else c[i] = raw[u].vc[i][0] >> (8 * (g >> 2));
                c[i] = (c[i] & 0x00ff00ffu) * 128u;
            }
            const Scale2 first(c[0]), second(c[1]);
#pragma unroll
            for (int w = 0; w < kVW; ++w) {
                const uint32_t *r0 = raw[u].v[0], *r1 = raw[u].v[1], *r2 = raw[u].v[2], *r3 = raw[u].v[3];
#pragma unroll
                for (int hl = 0; hl < 2; ++hl) {   // channels 0 .. 3 and 4 .. 7 of eight
                    uint32_t x[4], y[4];
                    unpack_q4(__byte_perm(r0[w], r1[w], hl ? 0x7632 : 0x5410), first, x);
                    unpack_q4(__byte_perm(r2[w], r3[w], hl ? 0x7632 : 0x5410), second, y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816(o[w * 4 + hl * 2][n], x[0], x[1], y[0], y[1], p[u][n][0], p[u][n][1]);
                        mma16816(o[w * 4 + hl * 2 + 1][n], x[2], x[3], y[2], y[3], p[u][n][0], p[u][n][1]);
                    }
                }
            }
        }
    }

    // the warps' results in shared memory, [head][channel]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = 8 * n + 2 * t + j;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], d);
            if (g == 0) {
                sm_m[warp][h] = m[n][j];
                sm_l[warp][h] = l[n][j];
            }
#pragma unroll
            for (int i = 0; i < kMT; ++i) {
                sm_o[warp][h][g * (D / 8) + 2 * i] = o[i][n][j];
                sm_o[warp][h][g * (D / 8) + 2 * i + 1] = o[i][n][j + 2];
            }
        }
    }
    __syncthreads();
    const long long part = ((long long)slice * a.splits + split) * a.group + h0;
    for (int i = tid; i < n_heads * (D / 4); i += kWarps * 32) {
        const int h = i / (D / 4), c = (i - h * (D / 4)) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w][h]);
        float den = 0.f, x[4] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (sm_m[w][h] == -INFINITY && sm_l[w][h] == 0.f) continue;   // no keys
            const float f = sm_m[w][h] == top ? 1.f : ex2_approx(sm_m[w][h] - top);
            den = fmaf(f, sm_l[w][h], den);
            const float4 y = *reinterpret_cast<const float4*>(&sm_o[w][h][c]);
            x[0] = fmaf(f, y.x, x[0]); x[1] = fmaf(f, y.y, x[1]);
            x[2] = fmaf(f, y.z, x[2]); x[3] = fmaf(f, y.w, x[3]);
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const float lse = den == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : (top - kLift) * 0.69314718056f) + logf(den);
        if (a.splits == 1) {
            const __nv_bfloat162 y[2] = {__floats2bfloat162_rn(x[0] * inv, x[1] * inv), __floats2bfloat162_rn(x[2] * inv, x[3] * inv)};
            *reinterpret_cast<uint2*>(a.out + (row0 + h) * D + c) = *reinterpret_cast<const uint2*>(y);
            if (c == 0 && a.lse) a.lse[row0 + h] = lse;
        } else {
            if (den != 0.f) *reinterpret_cast<float4*>(a.po + (part + h) * D + c) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            if (c == 0) a.plse[part + h] = lse;
        }
    }
}

// Key ranges per slice and their length: enough CTAs for four per SM four times over, of at least 128 keys.
static int q4_ranges(const AttnArgs& a, int* chunk) {
    const int head_tiles = (a.group + 15) / 16;
    const long long items = a.BH / a.group * head_tiles, want = (16LL * sm_count() + items - 1) / items;
    long long c = (a.L + want - 1) / want;
    if (c < 128) c = 128;
    if (want > 1 && c < 512 && items * ((a.L + 511) / 512) >= 4LL * sm_count()) c = 512;
    c = (c + 127) / 128 * 128;
    *chunk = (int)c;
    return (int)((a.L + c - 1) / c);
}
size_t attn_decode_q4_workspace(const AttnArgs& a) {
    int chunk;
    const size_t n = (size_t)q4_ranges(a, &chunk);
    return n > 1 ? align256((size_t)a.BH * n * a.D * 4) + align256((size_t)a.BH * n * 4) : 0;
}

template <int D, int NT>
static cudaError_t launch_q4(const AttnArgs& a, const CacheQ4& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    DecodeQ4Args g = {};
    g.q = (const __nv_bfloat16*)a.q;
    g.kc = (const unsigned char*)c.k; g.vc = (const unsigned char*)c.v;
    g.table = table; g.lens = lens;
    g.L = a.L; g.hkv = c.hkv; g.group = a.group; g.head_tiles = (a.group + 8 * NT - 1) / (8 * NT);
    g.n_pages = c.n_pages; g.page = c.page_size; g.max_pages = max_pages;
    g.splits = q4_ranges(a, &g.chunk);
    g.scale_log2 = a.scale * 1.4426950408889634f;
    g.out = (__nv_bfloat16*)a.out; g.lse = a.lse;
    g.po = (float*)ws;
    g.plse = (float*)((unsigned char*)ws + align256((size_t)a.BH * g.splits * D * 4));
    const long long ctas = a.BH / a.group * g.head_tiles * g.splits;
    if (ctas >= (1LL << 31)) return cudaErrorInvalidValue;
    {
        LaunchScope ls(K_DECODE_Q4, st);
        const cudaError_t e = launch_overlapped(attn_decode_q4_kernel<D, NT>, (unsigned)ctas, kWarps * 32, 0, st, g);
        if (e != cudaSuccess) return e;
    }
    return g.splits > 1 ? attn_decode_merge(a, g.po, g.plse, g.splits, st) : cudaSuccess;
}
cudaError_t attn_decode_q4(const AttnArgs& a, const CacheQ4& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    if (a.D == 128) return a.group <= 8 ? launch_q4<128, 1>(a, c, table, lens, max_pages, ws, st) : launch_q4<128, 2>(a, c, table, lens, max_pages, ws, st);
    return a.group <= 8 ? launch_q4<64, 1>(a, c, table, lens, max_pages, ws, st) : launch_q4<64, 2>(a, c, table, lens, max_pages, ws, st);
}

}  // namespace ttk
