// Single-query attention over the 4-bit key/value cache: out = softmax(scale q K^T) V with K, V = (n - 8) s.
//
// A key and key/value head are 2 (D / 2 + D / 32) bytes, at D = 128 136 of them for 256 values.  At the measured copy rate an SM
// gets 23 bytes a cycle, so it has 5.9 cycles for those 256 values: what bounds this next to HBM is the instructions that turn
// nibbles into operands.  Operands that are made in registers go to mma.sync, whose accumulators (16 x 8) a group of up to eight
// query heads fills; tcgen05 would want them in shared or tensor memory, 512 more bytes a key.
//
// Both products are m16n8k16 in halves with 32-bit sums (2.0 cycles per SM each; the 8-bit forms of mma.sync are made of these).  A lane
// reads exactly the nibbles that are its elements of the operand, and the order of channels within a product is chosen so that they are
// neighbours of one scale.  With 0x6400 above it a nibble is the half 1024 + n, or 1024 + 16 n four bits up, so a mask makes two halves and
// one fused multiply-add by the scale's multiples (n - 8) s / 16, or (n - 8) s, of them: exactly, for s has four significant bits and
// n - 8 four.  (Masks alone, without that, give n: for q with an outlier the -8 sum q then cancels in the tensor core's sums.)
//   S^T [16 keys x 8 heads] += K [16 keys x 16 channels] Q^T: lane (g, t) of a warp (g = lane / 4, t = lane % 4) has of keys g and g + 8 the
//     quarter t of the channels; q, its exponent moved so that a bf16 value down to 2^-27 of the head's largest is exact in half, is 16 times
//     higher for the channels whose keys are s / 16.
//   O^T [16 channels x 8 heads] += V^T [16 channels x 16 keys] P^T: lane (g, t) has of keys 2t, 2t + 1, 2t + 8, 2t + 9 the eighth g of the
//     channels, two keys beside each other in a word (a permute), and so its part of the result is D / 8 neighbouring channels of heads 2t
//     and 2t + 1; the rows of s / 16 are made good at the end.
//
// Softmax is online in base 2; the reference is raised, for all of a warp's heads, when a score passes it by 2^kSlack, and P is taken
// 2^kLift higher, up to 2^15: rounded to half it is off by 2^-11 of itself (bf16: 2^-8) down to 2^-24 of the row's largest, and by
// 2^-35 of that below.  Accumulators are 32-bit.
//
// A warp takes every fourth 32 keys of its CTA's range through a ring of its own in shared memory (cp.async, kDepth steps of 32 keys; no
// barrier between warps until the end); four warps and then the ranges are merged.
#include "cache_q4.cuh"
#include "sm100_ptx.cuh"

namespace ttk {
using namespace sm100;

namespace {

constexpr int kWarps = 4, kTile = 32, kDepth = 3;   // a step of a warp: 32 keys, two accumulator tiles of 16
constexpr float kSlack = 5.f, kLift = 10.f, kNone = -3e38f;   // (kNone: no score yet; above every finite one that counts as such)

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void copy16(uint32_t saddr, const void* p, bool some) {   // 16 bytes, or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(p), "r"(some ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[N], const unsigned char* p) {
    if (N == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x; w[1 % N] = x.y; w[2 % N] = x.z; w[3 % N] = x.w;
    } else if (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x; w[1 % N] = x.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
__device__ __forceinline__ half2 as_half2(uint32_t x) { return *reinterpret_cast<half2*>(&x); }
__device__ __forceinline__ uint32_t bits(half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// What two codes, times 128 in the halves of a word, make of nibbles: s8 = half(code << 7) = 8 s.  The codes that are written (and NaN) leave
// every constant finite and exact: 9 s8 <= 64512, and 129 / 16 times four significant bits has eleven.
struct Scale2 {
    half2 mul, even, odd;
    __device__ __forceinline__ explicit Scale2(uint32_t codes_times_128) {
        const half2 s8 = as_half2(codes_times_128);
        mul = __hmul2(s8, __float2half2_rn(1.f / 128));
        even = __hmul2(s8, __float2half2_rn(-129.f / 16));
        odd = __hmul2(s8, __float2half2_rn(-9.f));
    }
    // nibbles in the lowest bits of x's halves: (1024 + n) s8 / 128 - 129 s8 / 16 = (n - 8) s / 16
    __device__ __forceinline__ uint32_t low(uint32_t x, uint32_t k1024) const { return bits(__hfma2(as_half2(masked<0x000f000fu>(x, k1024)), mul, even)); }
    // four bits higher: (1024 + 16 n) s8 / 128 - 9 s8 = (n - 8) s
    __device__ __forceinline__ uint32_t high(uint32_t x, uint32_t k1024) const { return bits(__hfma2(as_half2(masked<0x00f000f0u>(x, k1024)), mul, odd)); }
    // (x & kMask) | k1024 in one instruction, which takes one constant: the other, 0x64006400, comes in a register that the compiler does not
    // see through
    template <uint32_t kMask>
    static __device__ __forceinline__ uint32_t masked(uint32_t x, uint32_t k1024) {
        uint32_t y;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "n"(kMask), "r"(k1024));
        return y;
    }
};

// 16 keys in a ring slot: rows of K, rows of V, K's codes, V's codes, 16-byte pieces in an order that keeps the reads off each
// other's banks.
template <int D>
struct Slot {
    static constexpr int kPieces = D / 32;   // of a row
    static constexpr int kV = 16 * D / 2, kKc = 2 * kV, kVc = kKc + 16 * (D / 32), kBytes = kVc + 16 * (D / 32);
    // K is read in whole rows, V as a quarter or half piece of every second row
    static __device__ __forceinline__ int k_at(int key, int piece) { return key * (D / 2) + piece * 16; }
    static __device__ __forceinline__ int v_at(int key, int piece) {
        if (D == 128) {
            const int line = key >> 1, p = (key & 1) * 4 + piece;
            return kV + line * 128 + ((p ^ ((line << 1 & 7) | (line >> 2 & 1))) << 4);
        }
        const int line = key >> 2, p = (key & 3) * 2 + piece;
        return kV + line * 128 + ((p ^ (line & 1) << 1) << 4);
    }
};

}  // namespace

struct DecodeQ4Args {
    const __nv_bfloat16* q;
    const unsigned char *kc, *vc;
    const int *table, *lens;
    int L, hkv, group, head_tiles, n_pages, page, max_pages, splits, chunk;
    float scale_log2;
    uint32_t k1024;   // 0x64006400, see Scale2
    __nv_bfloat16* out;   // splits == 1
    float* lse;           // may be null then
    float *po, *plse;     // splits > 1: normalised rows [slice, split, group, D] and log-sum-exps
};

template <int D, int NT>
constexpr int q4_smem() {
    const int ring = kWarps * kDepth * 2 * Slot<D>::kBytes, merge = kWarps * 8 * NT * (D + 4 + 2) * 4;
    return ring > merge ? ring : merge;
}

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 4 : D == 64 ? 3 : 2) attn_decode_q4_kernel(const DecodeQ4Args a) {
    constexpr int kHeads = 8 * NT, kG = D / 32, kVW = D / 64, kMT = D / 16;
    using S = Slot<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp_idx(), g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % a.splits, item = blockIdx.x / a.splits, tile = item % a.head_tiles, slice = item / a.head_tiles;
    const int b = slice / a.hkv, hk = slice - b * a.hkv, h0 = tile * kHeads, n_heads = min(kHeads, a.group - h0);
    const uint32_t k1024 = a.k1024;
    const uint32_t ring = smem_u32(smem) + warp * (kDepth * 2 * S::kBytes);
    grid_let_next_start();
    grid_wait_for_previous();
    const int len = a.lens ? min(max(__ldg(a.lens + b), 0), a.L) : a.L;
    const int k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
    const long long row0 = (long long)slice * a.group + h0;   // the tile's first query head

    // 16 keys lie in one page.  Lane i looks up where the i-th 16 keys of a batch are: the byte of their first row, or -1, and their row in
    // the page.
    const int n_sub = k1 > k0 ? ((k1 - k0 + kTile - 1) / kTile + kWarps - 1 - warp) / kWarps * 2 : 0;   // this warp's 16-key tiles
    auto first_key = [&](int sub) { return k0 + ((sub >> 1) * kWarps + warp) * kTile + (sub & 1) * 16; };
    long long at_now;
    int row_now;
    auto look_up = [&](int sub) {
        const int key = first_key(sub);
        at_now = -1;
        row_now = 0;
        if (sub < n_sub && key < k1) {
            const int col = key / a.page;
            const int page = !a.table ? b : col < a.max_pages ? __ldg(a.table + (long long)b * a.max_pages + col) : -1;
            if (page >= 0 && page < a.n_pages) {
                row_now = key - col * a.page;
                at_now = ((long long)page * a.hkv + hk) * ((long long)a.page * q4_row_bytes(D)) + row_now * (D / 2);
            }
        }
    };
    look_up(lane);
    // Pieces of a slot are numbered [K rows][V rows]; a lane copies every 32nd, and the first lanes the codes.
    constexpr int kCopies = 16 * S::kPieces / 32, kCodes = D / 32;   // per tensor; 16-byte pieces of codes
    uint32_t to_k[kCopies], to_v[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int piece = lane + 32 * i;
        to_k[i] = S::k_at(piece / S::kPieces, piece % S::kPieces);
        to_v[i] = S::v_at(piece / S::kPieces, piece % S::kPieces);
    }
    const unsigned char *from_k = a.kc + lane * 16, *from_v = a.vc + lane * 16;
    const unsigned char* from_codes = (lane < kCodes ? a.kc : a.vc) + a.page * (D / 2) + lane % kCodes * 16;
    // Both tiles of a step into the slots at `slot`: bits of those that have keys.
    auto fetch = [&](int sub, uint32_t slot) -> unsigned {
        unsigned has = 0;
        if (sub < n_sub) {
            if ((sub & 31) == 0 && sub > 0) look_up(sub + lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const long long at = __shfl_sync(0xffffffffu, at_now, (sub + j) & 31);
                const int row = __shfl_sync(0xffffffffu, row_now, (sub + j) & 31);
                const bool some = at >= 0;
                const uint32_t to = slot + j * S::kBytes;
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    copy16(to + to_k[i], from_k + at + 512 * i, some);
                    copy16(to + to_v[i], from_v + at + 512 * i, some);
                }
                if (lane < 2 * kCodes) copy16(to + S::kKc + lane * 16, from_codes + at - row * (D / 2 - D / 32), some);
                has |= some ? 1u << j : 0u;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return has;
    };
    unsigned has[kDepth];   // of the step at hand and those on their way
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) has[i] = fetch(2 * i, ring + i * 2 * S::kBytes);

    // query heads as the B operand: lane (g, t) has head g's quarter t of the channels, pairs (i, i + 4) of eight
    uint32_t qf[NT][kG][4];
    float to_log2[NT][2];   // the scores' factor of heads 2t and 2t + 1
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float x[kG][8], top = 0.f;
#pragma unroll
        for (int i = 0; i < kG; ++i) {
            const uint4 w = g + 8 * n < n_heads ? __ldg(reinterpret_cast<const uint4*>(a.q + (row0 + g + 8 * n) * D + t * (D / 4)) + i) : make_uint4(0, 0, 0, 0);
            const uint32_t y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][2 * j] = __uint_as_float(y[j] << 16);
                x[i][2 * j + 1] = __uint_as_float(y[j] & 0xffff0000u);
                top = fmaxf(top, fmaxf(fabsf(x[i][2 * j]), fabsf(x[i][2 * j + 1])));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the head's largest value to 2^10 .. 2^11 (infinities stay)
        const int e = (int)(__float_as_uint(top) >> 23) - 127, up = top > 0.f && e < 128 ? min(max(10 - e, -100), 100) : 0;
        const float f = __uint_as_float((unsigned)(up + 127) << 23), back = __uint_as_float((unsigned)(127 - up) << 23);
#pragma unroll
        for (int i = 0; i < kG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float by = j & 1 ? f : 16 * f;
                qf[n][i][j] = bits(__floats2half2_rn(x[i][j] * by, x[i][j + 4] * by));
            }
#pragma unroll
        for (int j = 0; j < 2; ++j) to_log2[n][j] = a.scale_log2 * __shfl_sync(0xffffffffu, back, (2 * t + j) * 4);
    }

    float o[kMT][NT][4], m[NT][2], l[NT][2];   // m: what a score is taken less; 2^-kLift of the reference
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][n][j] = 0.f;
        m[n][0] = m[n][1] = kNone;
        l[n][0] = l[n][1] = 0.f;
    }
    // where this lane reads in a slot
    uint32_t v_from[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v_from[i] = S::v_at(2 * t + (i & 1) + (i >> 1) * 8, g * (D / 16) / 16) + g * (D / 16) % 16;

    uint32_t at_slot = 0, free_slot = (kDepth - 1) * 2 * S::kBytes;   // of the step at hand, and of the one before it
    for (int sub = 0; sub < n_sub; sub += 2) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
        __syncwarp();
        const unsigned char* slot = smem + warp * (kDepth * 2 * S::kBytes) + at_slot;
        const unsigned here = has[0];
#pragma unroll
        for (int i = 0; i + 1 < kDepth; ++i) has[i] = has[i + 1];
        has[kDepth - 2] = fetch(sub + 2 * (kDepth - 1), ring + free_slot);   // every lane has left that slot
        free_slot = at_slot;
        at_slot = at_slot == (kDepth - 1) * 2 * S::kBytes ? 0 : at_slot + 2 * S::kBytes;
        // scores
        float s[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned char* from = slot + u * S::kBytes;
            uint32_t x[2][kG];
#pragma unroll
            for (int r = 0; r < 2; ++r) lds(x[r], from + (g + 8 * r) * (D / 2) + t * (D / 8));
            const Scale2 lo(from[S::kKc + g * (D / 32) + t * (D / 32) / 4] * 0x00800080u),
                hi(from[S::kKc + (g + 8) * (D / 32) + t * (D / 32) / 4] * 0x00800080u);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[u][n][j] = 0.f;
#pragma unroll
            for (int w = 0; w < kG; ++w) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // channels 0, 4 and 1, 5 of eight, then 2, 6 and 3, 7
                    const uint32_t y0 = x[0][w] >> 8 * h, y1 = x[1][w] >> 8 * h;
                    const uint32_t a0 = lo.low(y0, k1024), a1 = hi.low(y1, k1024), a2 = lo.high(y0, k1024), a3 = hi.high(y1, k1024);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(s[u][n], a0, a1, a2, a3, qf[n][w][2 * h], qf[n][w][2 * h + 1]);
                }
            }
        }
        // V's codes of keys 2t, 2t + 1 and 2t + 8, 2t + 9
        uint32_t vc[2][2][kVW];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) lds(vc[u][i], slot + u * S::kBytes + S::kVc + (2 * t + 8 * i) * (D / 32));
        // keys behind the range, or without a page: no score, and scales of 0 so that what lies there does not meet P = 0
        if (first_key(sub) + kTile > k1 || here != 3) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int left = here >> u & 1 ? k1 - first_key(sub + u) : 0;   // keys of these 16
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (g + (j >> 1) * 8 >= left) s[u][n][j] = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = 2 * t + 8 * i;
                    if (D == 128) {
                        if (key >= left) vc[u][i][0] = 0;
                        if (key + 1 >= left) vc[u][i][kVW - 1] = 0;
                    } else {
                        if (key >= left) vc[u][i][0] = 0;
                        else if (key + 1 >= left) vc[u][i][0] &= 0xffffu;
                    }
                }
            }
        }
        // the maximum, where a score passes it by 2^kSlack
        bool raise = false;
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[n][j] = fmaxf(fmaxf(s[0][n][j], s[0][n][j + 2]), fmaxf(s[1][n][j], s[1][n][j + 2])) * to_log2[n][j];
                raise = raise || top[n][j] > m[n][j] + (kLift + kSlack);
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
                    const float to = fmaxf(m[n][j], x - kLift), f = ex2_approx(m[n][j] - to);
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
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = ex2_approx(fmaf(s[u][n][2 * i], to_log2[n][0], -m[n][0])), y = ex2_approx(fmaf(s[u][n][2 * i + 1], to_log2[n][1], -m[n][1]));
                    l[n][0] += x;
                    l[n][1] += y;
                    p[u][n][i] = transposed8x8(bits(__floats2half2_rn(x, y)));
                }
            }
        }
        // O^T
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // the two keys' codes of the lane's group of channels, times 128, in the halves of a word
            uint32_t c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (D == 128) c[i] = __byte_perm(vc[u][i][0], vc[u][i][kVW - 1], (g >> 1) | (4 + (g >> 1)) << 8);
                else c[i] = vc[u][i][0] >> (8 * (g >> 2));
                c[i] = (c[i] & 0x00ff00ffu) * 128u;
            }
            const Scale2 first(c[0]), second(c[1]);
            uint32_t r[4][kVW];
#pragma unroll
            for (int i = 0; i < 4; ++i) lds(r[i], slot + u * S::kBytes + v_from[i]);
#pragma unroll
            for (int w = 0; w < kVW; ++w) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {   // byte j: channels 2j and 2j + 1 of the word's eight
                    const uint32_t sel = 0x0400u + 0x0101u * j;
                    const uint32_t x = __byte_perm(r[0][w], r[1][w], sel), y = __byte_perm(r[2][w], r[3][w], sel);
                    const uint32_t a0 = first.low(x, k1024), a1 = first.high(x, k1024), a2 = second.low(y, k1024), a3 = second.high(y, k1024);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[w * 4 + j][n], a0, a1, a2, a3, p[u][n][0], p[u][n][1]);
                }
            }
        }
    }

    // the warps' results in shared memory, [head][channel], over the rings
    float* sm_o = reinterpret_cast<float*>(smem);
    float* sm_m = sm_o + kWarps * kHeads * (D + 4);
    float* sm_l = sm_m + kWarps * kHeads;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = 8 * n + 2 * t + j, at = warp * kHeads + h;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], d);
            if (g == 0) {
                sm_m[at] = m[n][j];
                sm_l[at] = l[n][j];
            }
#pragma unroll
            for (int i = 0; i < kMT; ++i)
                *reinterpret_cast<float2*>(sm_o + at * (D + 4) + g * (D / 8) + 2 * i) = make_float2(16.f * o[i][n][j], o[i][n][j + 2]);
        }
    }
    __syncthreads();
    const long long part = ((long long)slice * a.splits + split) * a.group + h0;
    for (int i = tid; i < n_heads * (D / 4); i += kWarps * 32) {
        const int h = i / (D / 4), c = (i - h * (D / 4)) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w * kHeads + h]);
        float den = 0.f, x[4] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = sm_m[w * kHeads + h], lw = sm_l[w * kHeads + h];
            if (lw == 0.f) continue;   // no keys
            const float f = mw == top ? 1.f : ex2_approx(mw - top);
            den = fmaf(f, lw, den);
            const float4 y = *reinterpret_cast<const float4*>(sm_o + (w * kHeads + h) * (D + 4) + c);
            x[0] = fmaf(f, y.x, x[0]); x[1] = fmaf(f, y.y, x[1]);
            x[2] = fmaf(f, y.z, x[2]); x[3] = fmaf(f, y.w, x[3]);
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const float lse = den == 0.f ? -INFINITY : top * 0.69314718056f + logf(den);
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
    g.k1024 = 0x64006400u;
    g.out = (__nv_bfloat16*)a.out; g.lse = a.lse;
    g.po = (float*)ws;
    g.plse = (float*)((unsigned char*)ws + align256((size_t)a.BH * g.splits * D * 4));
    const long long ctas = a.BH / a.group * g.head_tiles * g.splits;
    if (ctas >= (1LL << 31)) return cudaErrorInvalidValue;
    {
        cudaError_t e = TT_ALLOW_SMEM((attn_decode_q4_kernel<D, NT>), (q4_smem<D, NT>()));
        if (e != cudaSuccess) return e;
        LaunchScope ls(K_DECODE_Q4, st);
        e = launch_overlapped(attn_decode_q4_kernel<D, NT>, (unsigned)ctas, kWarps * 32, q4_smem<D, NT>(), st, g);
        if (e != cudaSuccess) return e;
    }
    return g.splits > 1 ? attn_decode_merge(a, g.po, g.plse, g.splits, st) : cudaSuccess;
}
cudaError_t attn_decode_q4(const AttnArgs& a, const CacheQ4& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    if (a.D == 128) return a.group <= 8 ? launch_q4<128, 1>(a, c, table, lens, max_pages, ws, st) : launch_q4<128, 2>(a, c, table, lens, max_pages, ws, st);
    return a.group <= 8 ? launch_q4<64, 1>(a, c, table, lens, max_pages, ws, st) : launch_q4<64, 2>(a, c, table, lens, max_pages, ws, st);
}

}  // namespace ttk
