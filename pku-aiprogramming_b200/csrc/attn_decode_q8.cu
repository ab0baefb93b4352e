// Single-query attention over the 8-bit key/value cache: out = softmax(scale q K^T) V, K and V e4m3 codes times 2^e, one e for 16 tokens of a head.
//
// HBM-bound: a key and key/value head are 2 D bytes and two 16ths of one.  Codes become halves, exactly, in registers (a conversion makes two), which
// go to mma.sync: its accumulators (16 x 8) a group of up to eight query heads fills; tcgen05 would want q in codes too, in several parts, and P.  A warp takes up to
// 16 query heads; a larger group reads the cache once for each 16.  Both products are m16n8k16 in halves with 32-bit sums, 16 keys of one exponent at a time:
//   S^T [16 keys x 8 heads] += K [16 keys x 16 channels] Q^T: lane (g, t) of a warp (g = lane / 4, t = lane % 4) has of keys g and g + 8 every fourth
//     16 channels, four for each product; q, its exponent moved so that a bf16 value down to 2^-31 of the head's largest is exact in half.
//   O^T [16 channels x 8 heads] += V^T [16 channels x 16 keys] W^T: lane (g, t) has of keys 2t, 2t + 1, 2t + 8, 2t + 9 the eighth g of the channels,
//     two keys beside each other in a word (a permute), and so its part of the result is D / 8 neighbouring channels of heads 2t and 2t + 1.
//
// The exponents: a score is s = q k 2^ek, and the weight of a value code is 2^(s + ev).  Softmax is online in base 2 with x = s + ev in the place of s, so that
// weights keep their eleven bits next to the largest one whatever the exponents are, and sums of 2^-ev times the weights, in 32 bits, are the
// denominators.  The reference is raised, for all of a warp's heads, when an x passes it by 2^kSlack, and weights are taken 2^kLift higher, up to 2^15:
// rounded to half they are off by 2^-11 of themselves down to 2^-24 of the row's largest, and by 2^-35 of that below.
//
// The keys are shared out among the warps as decode_parts.cuh says; a warp streams its part through a ring of its own in shared memory (cp.async, kDepth steps,
// on into the next slice's keys where one ends).  In a slot 16 bytes of a row lie where neither product's reads meet in a bank.  No warp waits for another, and
// results do not depend on timing.
//
// Measured: 64 sequences of 4096 to 8192 keys, 32 heads on 8 of 128, 143 us, 5.7 TB/s (a copy runs at 6.6): beyond some 11 us, which are the chain lengths, page, exponents,
// keys at the start, one step more for some warps than for others, and the merge, a byte costs what it does at 6.2 TB/s.  16 heads on 16 of 64, 0 to 4096 keys,
// 48 us, 4.1 TB/s; 2 sequences of 120,000 keys, 32 heads on 2, 36 us, 3.6 TB/s of 128 MB.  Issue slots are a third to two fifths busy.
#include "cache_q8.cuh"
#include "decode_parts.cuh"
#include "sm100_ptx.cuh"

namespace ttk {
using namespace sm100;

namespace {

constexpr int kWarps = 4, kTile = 32, kDepth = 3;   // a step of a warp: 32 keys, two blocks of 16
constexpr float kSlack = 5.f, kLift = 10.f, kNone = -3e38f;   // (kNone: no score yet; above every finite one that counts as such)

// CTAs per SM: what their registers and rings leave room for.  D = 128: 2 (64 sequences of 4096 to 8192 keys, 8 heads, 143 us); 3 need rings of two steps and spill
// (164; 2 with such rings 148).  CTAs of three warps take 150 us, of two 158.
constexpr int q8_ctas_per_sm(int D, int NT) { return D == 128 ? 2 : NT == 1 ? 4 : 3; }
template <int D>
struct Q8Slot {   // 16 keys: rows of K, rows of V
    static constexpr int kV = 16 * D, kBytes = 2 * kV;
};
template <int D>
constexpr int q8_smem() { return kWarps * kDepth * 2 * Q8Slot<D>::kBytes; }

}  // namespace

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, q8_ctas_per_sm(D, NT)) attn_decode_q8_kernel(const PartsArgs a) {
    constexpr int kHeads = 8 * NT, kChunks = D / 64, kVW = D / 32, kMT = D / 16;   // 16 bytes of K, words of V, product tiles of a lane
    using S = Q8Slot<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = uniform_warp_idx(), g = lane >> 2, t = lane & 3;
    const unsigned char* ring = smem + warp * (kDepth * 2 * S::kBytes);
    const unsigned w_all = gridDim.x * kWarps, w = blockIdx.x + gridDim.x * warp, per_b = a.hkv * a.head_tiles;   // few parts: on different SMs
    grid_let_next_start();
    grid_wait_for_previous();

    PartsCursor<kTile> now{0, 0, 0};   // of the step at hand
    unsigned x0;                       // the part's first step, and how many it has
    int n;
    if (!parts_find<kTile, D, kHeads>(a, w, w_all, lane, &now, &x0, &n)) return;

    // 16 keys lie in one page.  Lane i looks up where the i-th 16 keys of a batch of 32 are, in units of 32 bytes (of which rows and pages are multiples), or
    // kNowhere; and their exponents, K's and V's, as the exponent bits of a float.
    constexpr unsigned kNowhere = 0xffffffffu;
    const long long page_bytes = q8_page_bytes(a.page, D);
    PartsCursor<kTile> ahead = now;
    unsigned rows_at, powers;
    auto look_up = [&](int sub) {   // sub: the lane's, a multiple of 32 for lane 0
        rows_at = kNowhere;
        powers = 127 | 127 << 16;
        if (sub < 2 * n) {
            const unsigned x = x0 + (sub >> 1);
            int step;
            ahead.to(a, per_b, x);
            const int slice = ahead.slice(x, &step), key = step * kTile + (sub & 1) * 16;
            if (key < ahead.len) {
                const int col = key / a.page;
                const int page = !a.table ? ahead.b : col < a.max_pages ? __ldg(a.table + (long long)ahead.b * a.max_pages + col) : -1;
                if (page >= 0 && page < a.n_pages) {
                    const int row = key - col * a.page;
                    const long long begin = ((long long)page * a.hkv + slice / a.head_tiles) * page_bytes, power = begin + (long long)a.page * D + row / kQ8Block;
                    rows_at = (unsigned)((begin + (long long)row * D) >> 5);
                    powers = (unsigned)(q8_exponent(a.kc[power]) + 127) | (unsigned)(q8_exponent(a.vc[power]) + 127) << 16;
                }
            }
        }
    };
    look_up(lane);
    // Where a lane's 16 bytes go: chunk c of row r of K to chunk c ^ 4 (r & 1) of its row (D = 128; at D = 64 two rows are a line and nothing moves), of V to
    // c ^ 2 (r / 2 & 3) of its line of 128 bytes.
    const unsigned char *from_k = a.kc + lane * 16, *from_v = a.vc + lane * 16;
    const uint32_t base = smem_u32(ring), into_k = base + (D == 128 ? (lane * 16) ^ ((lane >> 3 & 1) << 6) : lane * 16),
                   into_v = base + S::kV + (D == 128 ? (lane * 16) ^ ((lane >> 4 & 1) << 5) : (lane * 16) ^ ((lane >> 3 & 3) << 5));
    // Both blocks of step i into the ring at byte `to`; two bits: those that have keys.  Their exponents go with them.
    auto fetch = [&](int i, uint32_t to, unsigned (&power)[2]) -> unsigned {
        unsigned has = 0;
        power[0] = power[1] = 0;
        if (i < n) {
            if ((i & 15) == 0 && i > 0) look_up(2 * i + lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const unsigned at = __shfl_sync(0xffffffffu, rows_at, (2 * i + j) & 31);
                power[j] = __shfl_sync(0xffffffffu, powers, (2 * i + j) & 31);
                if (at != kNowhere) {
                    const uint32_t slot = to + j * S::kBytes;
                    const unsigned char *k = from_k + (unsigned long long)at * 32, *v = from_v + (unsigned long long)at * 32;
#pragma unroll
                    for (int c = 0; c < S::kV; c += 512) {
                        copy16(slot + into_k + c, k + c);
                        copy16((slot + into_v + c) ^ (D == 128 && (c & 512) ? 64u : 0u), v + c);
                    }
                    has |= 1u << j;
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return has;
    };
    unsigned has[kDepth], power[kDepth][2];   // of the step at hand and those on their way
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) has[i] = fetch(i, i * 2 * S::kBytes, power[i]);
    uint32_t at_slot = 0, free_slot = (kDepth - 1) * 2 * S::kBytes;   // of the step at hand, and of the one before it
    // where this lane reads in a slot: keys g and g + 8 of K (the second chunk at D = 128 is 64 bytes to one side or the other), key 2t of V
    const int k_from = g * D + (D == 128 ? (t * 16) ^ ((g & 1) << 6) : t * 16);
    const int v_from = S::kV + (D == 128 ? 2 * t * D + ((g * 16) ^ (t << 5)) : 2 * t * D + ((g * 8) ^ (t << 5)));

    for (int i = 0; i < n;) {   // slice by slice
        int step;
        now.to(a, per_b, x0 + i);
        const int slice_b = now.slice(x0 + i, &step), tile = slice_b % a.head_tiles;
        const long long slice = (long long)now.b * per_b + slice_b;
        const int h0 = tile * kHeads, n_heads = min(kHeads, a.group - h0), in_slice = (int)parts_steps<kTile>(now.len), end = min(n, i + in_slice - step);
        const bool whole = step == 0 && end - i == in_slice;
        const long long row0 = ((long long)now.b * a.hkv + slice_b / a.head_tiles) * a.group + h0;   // the tile's first query head

        // query heads as the B operand: lane (g, t) has of head g channels 16 t .. and 64 + 16 t .., pairs of four for each product
        uint32_t qf[NT][kChunks * 4][2];
        float to_log2[NT][2];   // the scores' factor of heads 2t and 2t + 1
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            float x[kChunks][16], top = 0.f;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 y4 = g + 8 * m < n_heads ? __ldg(reinterpret_cast<const uint4*>(a.q + (row0 + g + 8 * m) * D + c * 64 + t * 16) + half) : make_uint4(0, 0, 0, 0);
                    const uint32_t y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float &lo = x[c][8 * half + 2 * j], &hi = x[c][8 * half + 2 * j + 1];
                        lo = __uint_as_float(y[j] << 16);
                        hi = __uint_as_float(y[j] & 0xffff0000u);
                        top = fmaxf(top, fmaxf(fabsf(lo), fabsf(hi)));
                    }
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // The head's largest value to 2^14 .. 2^15 (infinities stay); half's last bit is 2^-24.  The move is held to 123, so that it and the move back are
            // normal floats.
            const int e = (int)(__float_as_uint(top) >> 23) - 127, up = top > 0.f && e < 128 ? min(14 - e, 123) : 0;
            const float f = __uint_as_float((unsigned)(up + 127) << 23), back = __uint_as_float((unsigned)(127 - up) << 23);
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const half2 y = __floats2half2_rn(x[c][4 * j + 2 * p] * f, x[c][4 * j + 2 * p + 1] * f);
                        qf[m][c * 4 + j][p] = *reinterpret_cast<const uint32_t*>(&y);
                    }
#pragma unroll
            for (int j = 0; j < 2; ++j) to_log2[m][j] = a.scale_log2 * __shfl_sync(0xffffffffu, back, (2 * t + j) * 4);
        }
        float o[kMT][NT][4], top_x[NT][2], above[NT][2];   // the reference, and what raises it
        uint64_t sums[NT];                                 // of 2^-ev times the weights, heads 2t and 2t + 1
#pragma unroll
        for (int m = 0; m < NT; ++m) {
#pragma unroll
            for (int c = 0; c < kMT; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[c][m][j] = 0.f;
            top_x[m][0] = top_x[m][1] = kNone;
            above[m][0] = above[m][1] = -INFINITY;
            sums[m] = 0;
        }
        int left = now.len - step * kTile;   // keys from the step at hand on
        for (; i < end; ++i, left -= kTile) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
            __syncwarp();
            const unsigned char* slot = ring + at_slot;
            const unsigned here = has[0];
            unsigned pw[2] = {power[0][0], power[0][1]};
#pragma unroll
            for (int k = 0; k + 1 < kDepth; ++k) {
                has[k] = has[k + 1];
                power[k][0] = power[k + 1][0];
                power[k][1] = power[k + 1][1];
            }
            has[kDepth - 2] = fetch(i + kDepth - 1, free_slot, power[kDepth - 2]);   // every lane has left that slot
            free_slot = at_slot;
            at_slot = at_slot == (kDepth - 1) * 2 * S::kBytes ? 0 : at_slot + 2 * S::kBytes;
            // scores
            float s[2][NT][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned char* from = slot + u * S::kBytes;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int at = c ? k_from ^ 64 : k_from;
                    const uint4 x4 = *reinterpret_cast<const uint4*>(from + at), y4 = *reinterpret_cast<const uint4*>(from + at + 8 * D);
                    const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t a0, a1, a2, a3;
                        q8_halves(x[j], a0, a2);
                        q8_halves(y[j], a1, a3);
#pragma unroll
                        for (int m = 0; m < NT; ++m) {
                            if (c + j == 0) mma_f16_first(s[u][m], a0, a1, a2, a3, qf[m][c * 4 + j][0], qf[m][c * 4 + j][1]);
                            else mma_f16(s[u][m], a0, a1, a2, a3, qf[m][c * 4 + j][0], qf[m][c * 4 + j][1]);
                        }
                    }
                }
            }
            const bool part = here != 3 || left < kTile;
            int keys[2];   // of the two blocks, where not all are there
#pragma unroll
            for (int u = 0; u < 2; ++u) keys[u] = here >> u & 1 ? left - 16 * u : 0;
            // x = s + ev
            float top[NT][2];
            bool raise = false;
            uint64_t x2[2][NT][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float pk = __uint_as_float((pw[u] & 0xffffu) << 23), ev = (float)((int)(pw[u] >> 16) - 127);
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    // (products of codes with half's values are 2^-33 .. 2^31 or 0, so that times the block's power is exact; the two factors' product may be infinite)
                    const uint64_t by = pack_f32x2(to_log2[m][0], to_log2[m][1]), block = pack_f32x2(pk, pk), more = pack_f32x2(ev, ev);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        x2[u][m][k] = fma_f32x2(mul_f32x2(pack_f32x2(s[u][m][2 * k], s[u][m][2 * k + 1]), block), by, more);
                        unpack_f32x2(x2[u][m][k], s[u][m][2 * k], s[u][m][2 * k + 1]);
                    }
                }
            }
            if (part) {   // keys that are not there, whatever their products are
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int m = 0; m < NT; ++m)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (g + k * 8 >= keys[u]) {
                                s[u][m][2 * k] = s[u][m][2 * k + 1] = -INFINITY;
                                x2[u][m][k] = pack_f32x2(-INFINITY, -INFINITY);
                            }
            }
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    top[m][j] = fmaxf(fmax3(s[0][m][j], s[0][m][j + 2], s[1][m][j]), s[1][m][j + 2]);
                    raise = raise || top[m][j] > above[m][j];
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    float f[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = top[m][j];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        const float to = fmaxf(top_x[m][j], x);
                        f[j] = ex2_approx(top_x[m][j] - to);
                        top_x[m][j] = to;
                        above[m][j] = __fadd_rd(to, kSlack);   // (beyond 2^24 the nearest may lie above to + kSlack, and a weight then beyond half)
#pragma unroll
                        for (int c = 0; c < kMT; ++c) {
                            o[c][m][j] *= f[j];
                            o[c][m][j + 2] *= f[j];
                        }
                    }
                    sums[m] = mul_f32x2(sums[m], pack_f32x2(f[0], f[1]));
                }
            }
            // weights, as the B operand
            uint32_t p[2][NT][2];
            const uint64_t lift = pack_f32x2(kLift, kLift);
#pragma unroll
            for (int m = 0; m < NT; ++m) {
                const uint64_t less = pack_f32x2(-top_x[m][0], -top_x[m][1]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float inv = __uint_as_float((254 - (pw[u] >> 16)) << 23);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x, y;
                        unpack_f32x2(add_f32x2(add_f32x2(x2[u][m][k], less), lift), x, y);
                        x = ex2_approx(x);
                        y = ex2_approx(y);
                        sums[m] = fma_f32x2(pack_f32x2(x, y), pack_f32x2(inv, inv), sums[m]);
                        const half2 z = __floats2half2_rn(x, y);
                        p[u][m][k] = transposed8x8(*reinterpret_cast<const uint32_t*>(&z));
                    }
                }
            }
            // O^T
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t r[4][kVW];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // (at D = 64 the odd row is the other half of the line)
                    const unsigned char* from = slot + u * S::kBytes + (k >> 1) * 8 * D + (D == 128 ? v_from + (k & 1) * D : v_from ^ (k & 1) << 6);
                    if constexpr (kVW == 4) {
                        const uint4 z = *reinterpret_cast<const uint4*>(from);
                        r[k][0] = z.x; r[k][1] = z.y; r[k][2] = z.z; r[k][3] = z.w;
                    } else {
                        const uint2 z = *reinterpret_cast<const uint2*>(from);
                        r[k][0] = z.x; r[k][1] = z.y;
                    }
                }
                if (part) {   // what lies behind the keys does not meet its weight of 0
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (2 * t + (k & 1) + (k >> 1) * 8 >= keys[u])
#pragma unroll
                            for (int j = 0; j < kVW; ++j) r[k][j] = 0;
                }
#pragma unroll
                for (int j = 0; j < kVW; ++j) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t sel = half ? 0x7362u : 0x5140u;   // channels 0 and 1, or 2 and 3, of two keys
                        const uint32_t x = __byte_perm(r[0][j], r[1][j], sel), y = __byte_perm(r[2][j], r[3][j], sel);
                        uint32_t a0, a1, a2, a3;
                        q8_halves(x, a0, a1);
                        q8_halves(y, a2, a3);
#pragma unroll
                        for (int m = 0; m < NT; ++m) mma_f16(o[j * 2 + half][m], a0, a1, a2, a3, p[u][m][0], p[u][m][1]);
                    }
                }
            }
        }

        // the part's result: lane (g, t) has channels g (D / 8) .. of heads 2t and 2t + 1
        const long long at_part = (w + slice) * a.part_rows;
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            float l[2];
            unpack_f32x2(sums[m], l[0], l[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int h = 8 * m + 2 * t + j;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], d);
                if (h >= n_heads) continue;
                const float den = l[j], inv = den == 0.f ? 0.f : 1.f / den;
                const float lse = den == 0.f ? -INFINITY : (top_x[m][j] - kLift) * 0.69314718056f + logf(den);
                float y[D / 8];
#pragma unroll
                for (int c = 0; c < kMT; ++c) {
                    y[2 * c] = o[c][m][j] * inv;
                    y[2 * c + 1] = o[c][m][j + 2] * inv;
                }
                if (whole) {
                    __nv_bfloat16* to = a.out + (row0 + h) * D + g * (D / 8);
#pragma unroll
                    for (int c = 0; c < D / 8; c += 8) {
                        const __nv_bfloat162 z[4] = {__floats2bfloat162_rn(y[c], y[c + 1]), __floats2bfloat162_rn(y[c + 2], y[c + 3]),
                                                     __floats2bfloat162_rn(y[c + 4], y[c + 5]), __floats2bfloat162_rn(y[c + 6], y[c + 7])};
                        *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(z);
                    }
                    if (g == 0 && a.lse) a.lse[row0 + h] = lse;
                } else {
                    float* to = a.po + (at_part + h) * D + g * (D / 8);
#pragma unroll
                    for (int c = 0; c < D / 8; c += 4) *reinterpret_cast<float4*>(to + c) = make_float4(y[c], y[c + 1], y[c + 2], y[c + 3]);
                    if (g == 0) a.plse[at_part + h] = lse;
                }
            }
        }
    }
}

// Whether every slice is one warp's, without a workspace and a second kernel: as long as one sequence takes no longer that way.  us so and in parts, one sequence and 64
// of 8 heads of 128, 128 keys 6.0 and 7.0, 7.8 and 10.8; 192 keys 7.4 and 7.4, 9.7 and 11.6; 256 keys 8.8 and 7.4, 11.5 and 13.1.
static bool q8_whole(const AttnArgs& a) { return a.L <= 6 * kTile; }
// CTAs: what an SM holds at once, fewer where there are not steps for their warps.
template <int NT>
static int q8_ctas(const AttnArgs& a, int head_tiles) {
    const long long slices = a.BH / a.group * head_tiles, steps = slices * ((a.L + kTile - 1) / kTile);
    const PartsShares shares((unsigned)steps, sm_count() * q8_ctas_per_sm(a.D, NT) * kWarps, (unsigned)slices);
    return (int)((shares.parts + kWarps - 1) / kWarps);
}
template <int NT>
static size_t q8_layout(const AttnArgs& a, PartsArgs* g, void* ws) {
    const int tiles = (a.group + 8 * NT - 1) / (8 * NT), rows = a.group < 8 * NT ? a.group : 8 * NT;
    if (g) g->head_tiles = tiles;
    if (q8_whole(a)) return 0;
    const size_t B = (size_t)(a.BH / a.H), parts = (size_t)q8_ctas<NT>(a, tiles) * kWarps + (size_t)(a.BH / a.group) * tiles;
    const size_t before = align256((B + 1) * 4), po = align256(parts * rows * a.D * 4);
    if (g) {
        g->before = (unsigned*)ws;
        g->po = (float*)((unsigned char*)ws + before);
        g->plse = (float*)((unsigned char*)ws + before + po);
        g->part_rows = rows;
    }
    return before + po + align256(parts * rows * 4);
}
size_t attn_decode_q8_workspace(const AttnArgs& a) { return a.group <= 8 ? q8_layout<1>(a, nullptr, nullptr) : q8_layout<2>(a, nullptr, nullptr); }

template <int D, int NT>
static cudaError_t launch_q8(const AttnArgs& a, const CacheQ8& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    PartsArgs g = {};
    g.q = (const __nv_bfloat16*)a.q;
    g.kc = (const unsigned char*)c.k; g.vc = (const unsigned char*)c.v;
    g.table = table; g.lens = lens;
    g.B = (int)(a.BH / a.H); g.L = a.L; g.hkv = c.hkv; g.group = a.group;
    g.n_pages = c.n_pages; g.page = c.page_size; g.max_pages = max_pages;
    g.scale_log2 = a.scale * 1.4426950408889634f;
    g.out = (__nv_bfloat16*)a.out; g.lse = a.lse;
    q8_layout<NT>(a, &g, ws);
    const bool whole = q8_whole(a);
    const int ctas = whole ? (int)((a.BH / a.group * g.head_tiles + kWarps - 1) / kWarps) : q8_ctas<NT>(a, g.head_tiles);
    cudaError_t e = TT_ALLOW_SMEM((attn_decode_q8_kernel<D, NT>), (q8_smem<D>()));
    if (e != cudaSuccess) return e;
    {
        LaunchScope ls(K_DECODE_Q8, st);
        e = launch_overlapped(attn_decode_q8_kernel<D, NT>, (unsigned)ctas, kWarps * 32, q8_smem<D>(), st, g);
        if (e != cudaSuccess || whole) return e;
    }
    return decode_parts_merge<D>(g, a, ctas * kWarps, st);
}
cudaError_t attn_decode_q8(const AttnArgs& a, const CacheQ8& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    if (a.D == 128) return a.group <= 8 ? launch_q8<128, 1>(a, c, table, lens, max_pages, ws, st) : launch_q8<128, 2>(a, c, table, lens, max_pages, ws, st);
    return a.group <= 8 ? launch_q8<64, 1>(a, c, table, lens, max_pages, ws, st) : launch_q8<64, 2>(a, c, table, lens, max_pages, ws, st);
}

}  // namespace ttk
