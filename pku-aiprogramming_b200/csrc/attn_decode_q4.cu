// Single-query attention over the 4-bit key/value cache: out = softmax(scale q K^T) V with K, V = (n - 8) s.
//
// A key and key/value head are 2 (D / 2 + D / 32) bytes, at D = 128 136 of them for 256 values.  At the measured copy rate an SM
// gets 23 bytes a cycle, so it has 5.9 cycles for those 256 values: next to HBM what counts is the instructions that turn
// nibbles into operands.  Operands that are made in registers go to mma.sync, whose accumulators (16 x 8) a group of up to eight
// query heads fills; tcgen05 would want them in shared or tensor memory, 512 more bytes a key.  A warp takes up to 16 query heads; a larger group reads and
// unpacks the cache once for each 16.
//
// Both products are m16n8k16 in halves with 32-bit sums (2.0 cycles per SM each; the 8-bit forms of mma.sync are made of these).  A lane
// reads exactly the nibbles that are its elements of the operand, and the order of channels within a product is chosen so that they are
// neighbours of one scale.  With 0x4800 above it a nibble is the half (1024 + n) / 128, or (1024 + 16 n) / 128 four bits up, so a mask makes two halves and
// one fused multiply-add by 8 s, which is the scale code's own bit pattern, (n - 8) s / 16, or (n - 8) s, of them: exactly, for s has four significant bits and
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
// All slices' keys, in steps of 32, make one sequence that is cut into equal parts, one for each warp on the GPU whatever the lengths are
// (a launch with a CTA per range of one slice ended on its last wave: 64 sequences of 4096 to 8192 106 us).  A warp sums the lengths,
// finds its part, and streams it through a ring of its own in shared memory (cp.async, kDepth steps, on into the next slice's keys where
// one ends; bulk copies of 1024 and 64 bytes were slower, 107 us for 95).  No warp waits for another.  A slice that one warp has to itself is written at once; of others each warp leaves
// a normalised result and its log-sum-exp, which a second kernel merges.  Results do not depend on timing.  Up to 128 keys a warp has a whole slice, and
// there is no second kernel.
//
// One B200, both kernels, replayed from a graph, three inputs in turn (bytes at the copy rate of 6.46 TB/s): 64 sequences of 4096 to 8192, 32 query on 8 key/value
// heads, D = 128 97.4 us (67.6); 48 of up to 4096, 16 on 16, D = 64 39.3 (16.2); two of 120,000 to 131,072, 32 on 2 32.4 (10.5); one of 5001, 32 on 8 10.0 (0.9).
// Counters of the first: 553 instructions per step of a warp, 336 of them unpacking and products, 138 cycles at four issues each where the bytes take 175;
// issue slots 56 % busy, ALU 47 %, half-precision multiply-adds 29 %, tensor pipe 26 %, at 1.75 GHz (power).  So no pipe bounds it but the order within a warp: it waits
// on its own arithmetic, and the loads do not run under all of it (without them 80.6 us, the loads alone 67, of 94).
#include "cache_q4.cuh"
#include "sm100_ptx.cuh"

namespace ttk {
using namespace sm100;

namespace {

constexpr int kWarps = 4, kTile = 32, kDepth = 3;   // a step of a warp: 32 keys, two accumulator tiles of 16
constexpr float kSlack = 5.f, kLift = 10.f, kNone = -3e38f;   // (kNone: no score yet; above every finite one that counts as such)
// References from here on (2^20): a score's last bit is 1/8 or more, so that adding a lift may round it to anything, and a fused multiply-add of it leaves what
// the reference's own product rounded off, which may be more than the exponential can take.  There is no lift then, the products are rounded first, and every
// step goes the way of those that raise the reference, where that is done, with 0 and 1 in its and the factor's place for the code behind.
constexpr float kFar = 1048576.f;

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
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void copy16(uint32_t saddr, const void* p) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(saddr), "l"(p) : "memory"); }
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
// every constant finite and exact: 9 s8 is at most 9 * 7168 = 64512 (half ends at 65504; the next code's 69120 would be infinite), and 129 / 16 times four significant bits has eleven.
static_assert(9 * ((8 + kQ4Top % 8) << (kQ4Top / 8 - 18)) <= 65504, "the largest code's constants are finite");
struct Scale2 {
    half2 s8, even, odd;
    __device__ __forceinline__ explicit Scale2(uint32_t codes_times_128) {
        s8 = as_half2(codes_times_128);
        even = __hmul2(s8, __float2half2_rn(-129.f / 16));
        odd = __hmul2(s8, __float2half2_rn(-9.f));
    }
    // nibbles in the lowest bits of x's halves: (1024 + n) / 128 s8 - 129 / 16 s8 = (n - 8) s / 16
    __device__ __forceinline__ uint32_t low(uint32_t x, uint32_t k8) const { return bits(__hfma2(as_half2(masked<0x000f000fu>(x, k8)), s8, even)); }
    // four bits higher: (1024 + 16 n) / 128 s8 - 9 s8 = (n - 8) s
    __device__ __forceinline__ uint32_t high(uint32_t x, uint32_t k8) const { return bits(__hfma2(as_half2(masked<0x00f000f0u>(x, k8)), s8, odd)); }
    // (x & kMask) | k8 in one instruction, which takes one constant: the other, 0x48004800, comes in a register that the compiler does not
    // see through
    template <uint32_t kMask>
    static __device__ __forceinline__ uint32_t masked(uint32_t x, uint32_t k8) {
        uint32_t y;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "n"(kMask), "r"(k8));
        return y;
    }
};

// 16 keys in a ring slot, each part as it lies in the page: rows of K, rows of V, K's codes, V's codes.
template <int D>
struct Slot {
    static constexpr int kRows = 16 * D / 2, kCodes = 16 * D / 32;
    static constexpr int kV = kRows, kKc = 2 * kRows, kVc = kKc + kCodes, kBytes = kVc + kCodes;
};

}  // namespace

struct DecodeQ4Args {
    const __nv_bfloat16* q;
    const unsigned char *kc, *vc;
    const int *table, *lens;
    int B, L, hkv, group, head_tiles, n_pages, page, max_pages;
    float scale_log2;
    uint32_t k8;    // 0x48004800, see Scale2
    __nv_bfloat16* out;
    float* lse;        // may be null
    // Workspace, unless every slice is one warp's (null then): steps before each batch entry [B + 1] (of one slice), and for every part of a slice that a warp does not have to itself the
    // normalised rows [part][part_rows][D] and log-sum-exps.  Parts are numbered warp + slice: one of the two grows from each to the next.
    unsigned* before;
    float *po, *plse;
    int part_rows;
};

// Of `total` steps warp w of `parts` has `per`, one more if it is among the first `rest`.  The host has batch x heads x L / 32 below 2^31, so counts
// fit 32 bits.
// At least two to a part where slices have 64 or more on average: the merge then takes longer than the second step; one sequence of 3000
// and eight heads 8.6 us for 9.1, of 16000 and one head 10.5 for 12.0; but 16 of 100 to 300 10.3 for 9.4, 64 of 10 to 100 11.4 for 10.2.
struct Q4Shares {
    unsigned parts, per, rest;
    __host__ __device__ __forceinline__ Q4Shares(unsigned total, unsigned warps, unsigned slices) {
        parts = total / 64 < slices ? total : (total + 1) / 2;
        parts = parts < 1 ? 1 : parts < warps ? parts : warps;
        per = total / parts;
        rest = total - per * parts;
    }
    __device__ __forceinline__ unsigned begin(unsigned w) const { return w * per + (w < rest ? w : rest); }
    __device__ __forceinline__ unsigned warp_of(unsigned x) const {
        const unsigned longer = rest * (per + 1);
        return x < longer ? x / (per + 1) : rest + (x - longer) / per;
    }
};

__device__ __forceinline__ int q4_len(const DecodeQ4Args& a, int b) { return a.lens ? min(max(__ldg(a.lens + b), 0), a.L) : a.L; }
__device__ __forceinline__ unsigned q4_steps(int len) { return (unsigned)(len + kTile - 1) / kTile; }

// A place in the sequence of steps: the batch entry it is in and where that one's steps begin.
struct Q4Cursor {
    int b, len;
    unsigned begin;
    __device__ __forceinline__ void to(const DecodeQ4Args& a, unsigned per_b, unsigned x) {   // x >= begin, below the end
        unsigned n;
        while (x - begin >= (n = q4_steps(len) * per_b)) {
            begin += n;
            len = q4_len(a, ++b);
        }
    }
    // the slice within the batch entry, and the step within the slice
    __device__ __forceinline__ int slice(unsigned x, int* step) const {
        const unsigned steps = q4_steps(len), s = (x - begin) / steps;
        *step = (int)(x - begin - s * steps);
        return (int)s;
    }
};

// What the registers hold.  D = 64, up to eight heads: 140.8 / 112.2 / 113.9 us for 64 sequences of 4096 to 8192 with three / four / five.  D = 128: four
// of 128 registers are no faster with 64 sequences (95.7 us for 97.5) and slower with one (14.0 for 12.2); up to 16 heads with their queries in shared
// memory, three of 162 registers: 33.8 for 33.0 with two of 131072, 29.0 for 27.3 with four of 7400.
constexpr int q4_ctas_per_sm(int D, int NT) { return NT == 1 ? (D == 64 ? 4 : 3) : D == 64 ? 3 : 2; }
template <int D, int NT>
constexpr int q4_smem() { return kWarps * kDepth * 2 * Slot<D>::kBytes; }

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, q4_ctas_per_sm(D, NT)) attn_decode_q4_kernel(const DecodeQ4Args a) {
    constexpr int kHeads = 8 * NT, kG = D / 32, kVW = D / 64, kMT = D / 16;
    using S = Slot<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    const int lane = threadIdx.x & 31, warp = uniform_warp_idx(), g = lane >> 2, t = lane & 3;
    const uint32_t k8 = a.k8;
    const unsigned char* ring = smem + warp * (kDepth * 2 * S::kBytes);
    const unsigned w_all = gridDim.x * kWarps, w = blockIdx.x + gridDim.x * warp, per_b = a.hkv * a.head_tiles;   // few parts: on different SMs
    grid_let_next_start();
    grid_wait_for_previous();

    Q4Cursor now{0, 0, 0};   // of the step at hand
    unsigned x0;             // the part's first step, and how many it has
    int n;
    if (!a.before) {   // a slice to a warp
        if (w >= a.B * per_b) return;
        now.b = w / per_b;
        now.len = q4_len(a, now.b);
        n = (int)q4_steps(now.len);
        x0 = (w - now.b * per_b) * n;   // (with the batch entry's own first step as 0)
        if (n == 0) {
            const int slice_b = w - now.b * per_b, h0 = slice_b % a.head_tiles * kHeads, n_heads = min(kHeads, a.group - h0);
            const long long row0 = ((long long)now.b * a.hkv + slice_b / a.head_tiles) * a.group + h0;
            for (int i = lane; i < n_heads * (D / 8); i += 32) reinterpret_cast<uint4*>(a.out + row0 * D)[i] = make_uint4(0, 0, 0, 0);
            if (lane < n_heads && a.lse) a.lse[row0 + lane] = -INFINITY;
            return;
        }
    } else {
        // the batch's steps, and where this warp's part begins
        unsigned sum = 0;
        for (int i = lane; i < a.B; i += 32) sum += q4_steps(q4_len(a, i));
        const unsigned total = __reduce_add_sync(0xffffffffu, sum) * per_b;
        const Q4Shares shares(total, w_all, a.B * per_b);
        if (w >= shares.parts) return;
        x0 = shares.begin(w);
        n = (int)(shares.begin(w + 1) - x0);
        const unsigned y = x0 / per_b;
        unsigned done = 0;
        int found = -1;
        for (int i = 0; i < a.B && (found < 0 || w == 0); i += 32) {
            const int len = i + lane < a.B ? q4_len(a, i + lane) : 0;
            unsigned to = q4_steps(len);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffffu, to, d);
                if (lane >= d) to += x;
            }
            to += done;
            if (w == 0 && i + lane < a.B) {   // for the merge
                a.before[i + lane + 1] = to;
                if (i + lane == 0) a.before[0] = 0;
            }
            const unsigned past = __ballot_sync(0xffffffffu, to > y);
            if (found < 0 && past) {
                const int at = __ffs(past) - 1;
                found = i + at;
                now.b = found;
                now.len = __shfl_sync(0xffffffffu, len, at);
                now.begin = (__shfl_sync(0xffffffffu, to, at) - q4_steps(now.len)) * per_b;
            }
            done = __shfl_sync(0xffffffffu, to, 31);
        }
        if (found < 0) return;   // no keys at all
    }

    // 16 keys lie in one page.  Lane i looks up where the i-th 16 keys of a batch of 32 are: the first row and its codes, in units of 32 bytes
    // (of which all of these are multiples), or kNowhere.
    constexpr unsigned kNowhere = 0xffffffffu;
    Q4Cursor ahead = now;
    unsigned rows_at, codes_at;
    auto look_up = [&](int sub) {   // sub: the lane's, a multiple of 32 for lane 0
        rows_at = codes_at = kNowhere;
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
                    const long long begin = ((long long)page * a.hkv + slice / a.head_tiles) * ((long long)a.page * q4_row_bytes(D));
                    rows_at = (unsigned)((begin + (long long)row * (D / 2)) >> 5);
                    codes_at = (unsigned)((begin + (long long)a.page * (D / 2) + row * (D / 32)) >> 5);
                }
            }
        }
    };
    look_up(lane);
    constexpr int kCodeCopies = S::kCodes / 16;   // lanes that copy codes of K, and of V
    const unsigned char *from_k = a.kc + lane * 16, *from_v = a.vc + lane * 16, *from_codes = (lane < kCodeCopies ? a.kc : a.vc) + lane % kCodeCopies * 16;
    const uint32_t into = smem_u32(ring) + lane * 16;
    // Both tiles of step i into the ring at byte `to`; two bits: those that have keys.
    auto fetch = [&](int i, uint32_t to) -> unsigned {
        unsigned has = 0;
        if (i < n) {
            if ((i & 15) == 0 && i > 0) look_up(2 * i + lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const unsigned at = __shfl_sync(0xffffffffu, rows_at, (2 * i + j) & 31), codes = __shfl_sync(0xffffffffu, codes_at, (2 * i + j) & 31);
                if (at != kNowhere) {
                    const uint32_t slot = into + to + j * S::kBytes;
                    const unsigned char *k = from_k + (unsigned long long)at * 32, *v = from_v + (unsigned long long)at * 32;
#pragma unroll
                    for (int c = 0; c < S::kRows; c += 512) {
                        copy16(slot + c, k + c);
                        copy16(slot + S::kV + c, v + c);
                    }
                    if (lane < 2 * kCodeCopies) copy16(slot + S::kKc, from_codes + (unsigned long long)codes * 32);
                    has |= 1u << j;
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return has;
    };
    unsigned has[kDepth];   // of the step at hand and those on their way
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) has[i] = fetch(i, i * 2 * S::kBytes);
    uint32_t at_slot = 0, free_slot = (kDepth - 1) * 2 * S::kBytes;   // of the step at hand, and of the one before it
    // where this lane reads in a slot: keys g and g + 8 of K, key 2t of V, codes of key g and of key 2t
    const int k_from = g * (D / 2) + t * (D / 8), v_from = S::kV + 2 * t * (D / 2) + g * (D / 16), kc_from = S::kKc + g * (D / 32) + t * (D / 32) / 4,
              vc_from = S::kVc + 2 * t * (D / 32);

    for (int i = 0; i < n;) {   // slice by slice
        int step;
        now.to(a, per_b, x0 + i);
        const int slice_b = now.slice(x0 + i, &step), tile = slice_b % a.head_tiles;
        const long long slice = (long long)now.b * per_b + slice_b;
        const int h0 = tile * kHeads, n_heads = min(kHeads, a.group - h0), in_slice = (int)q4_steps(now.len), end = min(n, i + in_slice - step);
        const bool whole = step == 0 && end - i == in_slice;
        const long long row0 = ((long long)now.b * a.hkv + slice_b / a.head_tiles) * a.group + h0;   // the tile's first query head

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
            // The head's largest value to 2^10 .. 2^11 (infinities stay).  e is -127 .. 127, so the move is -117 or more; it ends at 123, where a value of
            // bf16, subnormal ones too, is a multiple of 2^-10.  All of f, 16 f and back are normal floats.
            const int e = (int)(__float_as_uint(top) >> 23) - 127, up = top > 0.f && e < 128 ? min(10 - e, 123) : 0;
            const float f = __uint_as_float((unsigned)(up + 127) << 23), back = __uint_as_float((unsigned)(127 - up) << 23);
#pragma unroll
            for (int i = 0; i < kG; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float by = j & 1 ? f : 16 * f;
                    qf[n][i][j] = bits(__floats2half2_rn(x[i][j] * by, x[i][j + 4] * by));
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)   // (not 0, which times the -inf of absent keys is no number; sums are below 2^31, so what it is held from is 0)
                to_log2[n][j] = fmaxf(a.scale_log2 * __shfl_sync(0xffffffffu, back, (2 * t + j) * 4), 1.1754944e-38f);
        }
        float o[kMT][NT][4], m[NT][2], above[NT][2];   // m: what a score is taken less, 2^-kLift of the reference; above: what raises it
        uint64_t sums[NT];                              // of P, heads 2t and 2t + 1
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < kMT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][n][j] = 0.f;
            m[n][0] = m[n][1] = kNone;
            above[n][0] = above[n][1] = -INFINITY;
            sums[n] = 0;
        }
        bool far = false;                    // whether a head's reference is kFar or more, the true ones and the factors in `kept` then (in local memory: rare)
        volatile float kept[NT][4];
        int left = now.len - step * kTile;   // keys from the step at hand on
        for (; i < end; ++i, left -= kTile) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
            __syncwarp();
            const unsigned char* slot = ring + at_slot;
            const unsigned here = has[0];
#pragma unroll
            for (int k = 0; k + 1 < kDepth; ++k) has[k] = has[k + 1];
            has[kDepth - 2] = fetch(i + kDepth - 1, free_slot);   // every lane has left that slot
            free_slot = at_slot;
            at_slot = at_slot == (kDepth - 1) * 2 * S::kBytes ? 0 : at_slot + 2 * S::kBytes;
            // scores
            float s[2][NT][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned char* from = slot + u * S::kBytes;
                uint32_t x[2][kG];
#pragma unroll
                for (int r = 0; r < 2; ++r) lds(x[r], from + k_from + r * 8 * (D / 2));
                const Scale2 lo(from[kc_from] * 0x00800080u), hi(from[kc_from + 8 * (D / 32)] * 0x00800080u);
#pragma unroll
                for (int w = 0; w < kG; ++w) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {   // channels 0, 4 and 1, 5 of eight, then 2, 6 and 3, 7
                        const uint32_t y0 = x[0][w] >> 8 * h, y1 = x[1][w] >> 8 * h;
                        const uint32_t a0 = lo.low(y0, k8), a1 = hi.low(y1, k8), a2 = lo.high(y0, k8), a3 = hi.high(y1, k8);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (w + h == 0) mma_f16_first(s[u][n], a0, a1, a2, a3, qf[n][w][2 * h], qf[n][w][2 * h + 1]);
                            else mma_f16(s[u][n], a0, a1, a2, a3, qf[n][w][2 * h], qf[n][w][2 * h + 1]);
                        }
                    }
                }
            }
            // V's codes of keys 2t, 2t + 1 and 2t + 8, 2t + 9
            uint32_t vc[2][2][kVW];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) lds(vc[u][i], slot + u * S::kBytes + vc_from + i * 8 * (D / 32));
            // keys behind the range, or without a page: no score, and scales of 0 so that what lies there does not meet P = 0
            if (here != 3 || left < kTile) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int keys = here >> u & 1 ? left - 16 * u : 0;   // of these 16
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (g + (j >> 1) * 8 >= keys) s[u][n][j] = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = 2 * t + 8 * i;
                        if (D == 128) {
                            if (key >= keys) vc[u][i][0] = 0;
                            if (key + 1 >= keys) vc[u][i][kVW - 1] = 0;
                        } else {
                            if (key >= keys) vc[u][i][0] = 0;
                            else if (key + 1 >= keys) vc[u][i][0] &= 0xffffu;
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
                    top[n][j] = fmaxf(fmax3(s[0][n][j], s[0][n][j + 2], s[1][n][j]), s[1][n][j + 2]);
                    raise = raise || top[n][j] > above[n][j];
                }
            }
            if (__any_sync(0xffffffffu, raise)) {
                if (far) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            m[n][j] = kept[n][j];
                            to_log2[n][j] = kept[n][2 + j];
                        }
                }
                bool here_far = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = top[n][j];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        const float y = __fmul_rn(x, to_log2[n][j]), to = fmaxf(m[n][j], fabsf(y) < kFar ? y - kLift : y);
                        f[j] = ex2_approx(m[n][j] - to);
                        m[n][j] = to;
                        above[n][j] = (to + (kLift + kSlack)) / to_log2[n][j];
                        here_far = here_far || (fabsf(to) >= kFar - 2 * kLift && to != kNone);
#pragma unroll
                        for (int c = 0; c < kMT; ++c) {
                            o[c][n][j] *= f[j];
                            o[c][n][j + 2] *= f[j];
                        }
                    }
                    sums[n] = mul_f32x2(sums[n], pack_f32x2(f[0], f[1]));
                }
                far = __any_sync(0xffffffffu, here_far);
                if (far) {   // see kFar
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int k = j; k < 4; k += 2) s[u][n][k] = __fadd_rn(__fmul_rn(s[u][n][k], to_log2[n][j]), -m[n][j]);
                            kept[n][j] = m[n][j];
                            kept[n][2 + j] = to_log2[n][j];
                            m[n][j] = 0.f;
                            to_log2[n][j] = 1.f;
                            above[n][j] = -INFINITY;
                        }
                }
            }
            // P^T as the B operand
            uint32_t p[2][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint64_t less = pack_f32x2(-m[n][0], -m[n][1]), by = pack_f32x2(to_log2[n][0], to_log2[n][1]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x, y;
                        unpack_f32x2(fma_f32x2(pack_f32x2(s[u][n][2 * k], s[u][n][2 * k + 1]), by, less), x, y);
                        x = ex2_approx(x);
                        y = ex2_approx(y);
                        sums[n] = add_f32x2(sums[n], pack_f32x2(x, y));
                        p[u][n][k] = transposed8x8(bits(__floats2half2_rn(x, y)));
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
                for (int k = 0; k < 4; ++k) lds(r[k], slot + u * S::kBytes + v_from + ((k & 1) + (k >> 1) * 8) * (D / 2));
#pragma unroll
                for (int w = 0; w < kVW; ++w) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {   // byte j: channels 2j and 2j + 1 of the word's eight
                        const uint32_t sel = 0x0400u + 0x0101u * j;
                        const uint32_t x = __byte_perm(r[0][w], r[1][w], sel), y = __byte_perm(r[2][w], r[3][w], sel);
                        const uint32_t a0 = first.low(x, k8), a1 = first.high(x, k8), a2 = second.low(y, k8), a3 = second.high(y, k8);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_f16(o[w * 4 + j][n], a0, a1, a2, a3, p[u][n][0], p[u][n][1]);
                    }
                }
            }
        }

        if (far) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) m[n][j] = kept[n][j];
        }
        // the part's result: lane (g, t) has channels g (D / 8) .. of heads 2t and 2t + 1
        const long long part = (w + slice) * a.part_rows;
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8) {
            float l[2];
            unpack_f32x2(sums[n8], l[0], l[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int h = 8 * n8 + 2 * t + j;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], d);
                if (h >= n_heads) continue;
                const float den = l[j], inv = den == 0.f ? 0.f : 1.f / den;
                const float lse = den == 0.f ? -INFINITY : m[n8][j] * 0.69314718056f + logf(den);
                float y[D / 8];
#pragma unroll
                for (int c = 0; c < kMT; ++c) {
                    y[2 * c] = 16.f * o[c][n8][j] * inv;
                    y[2 * c + 1] = o[c][n8][j + 2] * inv;
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
                    float* to = a.po + (part + h) * D + g * (D / 8);
#pragma unroll
                    for (int c = 0; c < D / 8; c += 4) *reinterpret_cast<float4*>(to + c) = make_float4(y[c], y[c + 1], y[c + 2], y[c + 3]);
                    if (g == 0) a.plse[part + h] = lse;
                }
            }
        }
    }
}

// kT threads per query head: zeros for a sequence without keys, nothing where one warp had the whole slice, else the sum of the parts' rows weighted
// by exp(log-sum-exp).  What bounds it is latency: the parts' places, then their log-sum-exps and the first rows at once; 3 to 6 us behind the other
// kernel.  Both kernels, with 32 / 128 / 256 / 512 threads a row: 7 parts of 3840 rows 18.3 / 22.8 / 31.2 / 51.3 us, 15 of 1280 rows 28.3 / 27.3 /
// 30.5 / 37.5, 28 of 512 rows 19.0 / 19.4 / 16.2 / 19.1, 222 of 32 rows 16.9 / 10.7 / 10.1 / 9.9, 1776 of 8 rows 116 / 36 / 24 / 17.5.
constexpr int kMergeParts = 1024;   // weights held at a time
template <int D, int kT>
__global__ void __launch_bounds__(kT == 32 ? 128 : kT) attn_decode_q4_merge_kernel(const DecodeQ4Args a, int heads, int rows_all, int w_all) {
    constexpr int kLanes = D / 4, kRows = kT / kLanes > 0 ? kT / kLanes : 1, kAhead = 4, kWeights = kT == 32 ? 32 : kMergeParts;
    static_assert(kT % kLanes == 0, "whole rows");
    __shared__ float sm_w[kT == 32 ? 4 : 1][kWeights], sm_o[kT == 32 ? 1 : kRows][D], sm_r[2][kT / 32];
    const int tid = threadIdx.x % kT, lane = tid & 31, mine = kT == 32 ? threadIdx.x / 32 : 0, row = kT == 32 ? blockIdx.x * 4 + mine : blockIdx.x;
    if (row >= rows_all) return;
    const int hq = row % heads, b = row / heads, group_tile = hq % a.group / a.part_rows, h = hq % a.group % a.part_rows;
    const int per_b = a.hkv * a.head_tiles, slice_b = hq / a.group * a.head_tiles + group_tile;
    auto barrier = [] {
        if (kT == 32) __syncwarp();
        else __syncthreads();
    };
    grid_wait_for_previous();
    grid_let_next_start();   // (before the wait the next call's CTAs crowd in among the first kernel's: 34.4 us for 27.7 with 32 sequences of up to 4000)
    const unsigned first = a.before[b], steps = a.before[b + 1] - first, total = a.before[a.B] * per_b;
    __nv_bfloat16* out = a.out + (long long)row * D;
    if (steps == 0) {
        for (int c = tid; c < D / 2; c += kT) reinterpret_cast<uint32_t*>(out)[c] = 0;
        if (tid == 0 && a.lse) a.lse[row] = -INFINITY;
        return;
    }
    const Q4Shares shares(total, w_all, a.B * per_b);
    const unsigned x = first * per_b + slice_b * steps;
    const int w0 = (int)shares.warp_of(x), n = (int)shares.warp_of(x + steps - 1) - w0 + 1;
    if (n == 1) return;
    const long long part = w0 + (long long)b * per_b + slice_b;
    const float* plse = a.plse + part * a.part_rows + h;
    const int r0 = tid / kLanes, col = tid % kLanes * 4;
    const float* rows = a.po + (part * a.part_rows + h) * D + col;
    float4 v[kAhead];
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k * kRows;
            v[k] = i < n ? *reinterpret_cast<const float4*>(rows + (long long)i * a.part_rows * D) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    load(r0);
    auto reduced = [&](float y, bool max, int at) {   // over the row's threads, `at` 0 or 1
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const float z = __shfl_xor_sync(0xffffffffu, y, d);
            y = max ? fmaxf(y, z) : y + z;
        }
        if (kT == 32) return y;
        if (lane == 0) sm_r[at][tid >> 5] = y;
        __syncthreads();
        y = sm_r[at][0];
#pragma unroll
        for (int i = 1; i < kT / 32; ++i) y = max ? fmaxf(y, sm_r[at][i]) : y + sm_r[at][i];
        return y;
    };
    float top = -INFINITY, den = 0.f;
    for (int i = tid; i < n; i += kT) top = fmaxf(top, plse[(long long)i * a.part_rows]);
    top = reduced(top, true, 0);
    if (top == -INFINITY) top = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = 0; base < n; base += kWeights) {
        const int end = min(base + kWeights, n);
        if (base) barrier();
        for (int i = base + tid; i < end; i += kT) {
            const float y = plse[(long long)i * a.part_rows], e = y == -INFINITY ? 0.f : expf(y - top);
            sm_w[mine][i - base] = e;
            den += e;
        }
        barrier();
        for (int i0 = base + r0; i0 < end; i0 += kAhead * kRows) {
            if (i0 != r0) load(i0);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kRows;
                const float f = i < end ? sm_w[mine][i - base] : 0.f;
                acc.x = fmaf(f, v[k].x, acc.x); acc.y = fmaf(f, v[k].y, acc.y);
                acc.z = fmaf(f, v[k].z, acc.z); acc.w = fmaf(f, v[k].w, acc.w);
            }
        }
    }
    if (kT != 32) *reinterpret_cast<float4*>(&sm_o[r0][col]) = acc;
    den = reduced(den, false, 1);   // (its barrier orders sm_o too)
    const float inv = den == 0.f ? 0.f : 1.f / den;
    if (kT == 32) {
#pragma unroll
        for (int d = 16; d >= kLanes; d >>= 1) {   // D = 64: two rows to a warp
            acc.x += __shfl_xor_sync(0xffffffffu, acc.x, d); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, d);
            acc.z += __shfl_xor_sync(0xffffffffu, acc.z, d); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, d);
        }
        const __nv_bfloat162 z[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
        if (r0 == 0) *reinterpret_cast<uint2*>(out + col) = *reinterpret_cast<const uint2*>(z);
    } else {
        for (int c = tid; c < D; c += kT) {
            float y = 0.f;
#pragma unroll
            for (int r = 0; r < kRows; ++r) y += sm_o[r][c];
            out[c] = __float2bfloat16_rn(y * inv);
        }
    }
    if (tid == 0 && a.lse) a.lse[row] = den == 0.f ? -INFINITY : top + logf(den);
}

// Whether every slice is one warp's, without a workspace and a second kernel: where the steps that a warp then has in a row take less time than the merge. From
// a graph / as calls, us, for the two kernels: 64 sequences of up to 20 keys, 32 on 8 heads, 4.9 / 5.7 for 7.0 / 8.3, of up to 60 6.1 / 5.6 for 9.4 / 10.0, of up to 100 7.6 / 8.4
// for 10.2 / 10.4, of up to 250 12.9 / 14.3 for 13.2 / 13.8, of up to 500 22.2 / 24.0 for 15.5 / 16.0; two of 200 8.2 / 8.7 for 7.4 / 8.2.
static bool q4_whole(const AttnArgs& a) { return a.L <= 4 * kTile; }
// CTAs: what an SM holds at once, fewer where there are not steps for their warps.
template <int NT>
static int q4_ctas(const AttnArgs& a, int head_tiles) {
    const long long slices = a.BH / a.group * head_tiles, steps = slices * ((a.L + kTile - 1) / kTile);
    const Q4Shares shares((unsigned)steps, sm_count() * q4_ctas_per_sm(a.D, NT) * kWarps, (unsigned)slices);
    return (int)((shares.parts + kWarps - 1) / kWarps);
}
template <int NT>
static size_t q4_layout(const AttnArgs& a, DecodeQ4Args* g, void* ws) {
    const int tiles = (a.group + 8 * NT - 1) / (8 * NT), rows = a.group < 8 * NT ? a.group : 8 * NT;
    if (g) g->head_tiles = tiles;
    if (q4_whole(a)) return 0;
    const size_t B = (size_t)(a.BH / a.H), parts = (size_t)q4_ctas<NT>(a, tiles) * kWarps + (size_t)(a.BH / a.group) * tiles;
    const size_t before = align256((B + 1) * 4), po = align256(parts * rows * a.D * 4);
    if (g) {
        g->before = (unsigned*)ws;
        g->po = (float*)((unsigned char*)ws + before);
        g->plse = (float*)((unsigned char*)ws + before + po);
        g->part_rows = rows;
    }
    return before + po + align256(parts * rows * 4);
}
size_t attn_decode_q4_workspace(const AttnArgs& a) { return a.group <= 8 ? q4_layout<1>(a, nullptr, nullptr) : q4_layout<2>(a, nullptr, nullptr); }

template <int D, int kT>
static cudaError_t launch_q4_merge(const DecodeQ4Args& g, const AttnArgs& a, int n_warps, cudaStream_t st) {
    constexpr int kRows = kT == 32 ? 4 : 1;
    LaunchScope ls(K_DECODE_MERGE, st);
    return launch_overlapped(attn_decode_q4_merge_kernel<D, kT>, (unsigned)((a.BH + kRows - 1) / kRows), kT * kRows, 0, st, g, a.H, (int)a.BH, n_warps);
}
template <int D, int NT>
static cudaError_t launch_q4(const AttnArgs& a, const CacheQ4& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    DecodeQ4Args g = {};
    g.q = (const __nv_bfloat16*)a.q;
    g.kc = (const unsigned char*)c.k; g.vc = (const unsigned char*)c.v;
    g.table = table; g.lens = lens;
    g.B = (int)(a.BH / a.H); g.L = a.L; g.hkv = c.hkv; g.group = a.group;
    g.n_pages = c.n_pages; g.page = c.page_size; g.max_pages = max_pages;
    g.scale_log2 = a.scale * 1.4426950408889634f;
    g.k8 = 0x48004800u;
    g.out = (__nv_bfloat16*)a.out; g.lse = a.lse;
    q4_layout<NT>(a, &g, ws);
    const bool whole = q4_whole(a);
    const int ctas = whole ? (int)((a.BH / a.group * g.head_tiles + kWarps - 1) / kWarps) : q4_ctas<NT>(a, g.head_tiles);
    cudaError_t e = TT_ALLOW_SMEM((attn_decode_q4_kernel<D, NT>), (q4_smem<D, NT>()));
    if (e != cudaSuccess) return e;
    {
        LaunchScope ls(K_DECODE_Q4, st);
        e = launch_overlapped(attn_decode_q4_kernel<D, NT>, (unsigned)ctas, kWarps * 32, q4_smem<D, NT>(), st, g);
        if (e != cudaSuccess || whole) return e;
    }
    // A warp for a row of up to a dozen parts, if all slices were of the greatest length; else as many threads as leave all rows in one wave.
    const int n_warps = ctas * kWarps;
    if (n_warps <= 12 * (a.BH / a.group) * g.head_tiles) return launch_q4_merge<D, 32>(g, a, n_warps, st);
    const long long room = sm_count() * 1024LL;
    if (a.BH * 512 <= room) return launch_q4_merge<D, 512>(g, a, n_warps, st);
    return a.BH * 256 <= room ? launch_q4_merge<D, 256>(g, a, n_warps, st) : launch_q4_merge<D, 128>(g, a, n_warps, st);
}
cudaError_t attn_decode_q4(const AttnArgs& a, const CacheQ4& c, const int* table, const int* lens, int max_pages, void* ws, cudaStream_t st) {
    if (a.D == 128) return a.group <= 8 ? launch_q4<128, 1>(a, c, table, lens, max_pages, ws, st) : launch_q4<128, 2>(a, c, table, lens, max_pages, ws, st);
    return a.group <= 8 ? launch_q4<64, 1>(a, c, table, lens, max_pages, ws, st) : launch_q4<64, 2>(a, c, table, lens, max_pages, ws, st);
}

}  // namespace ttk
