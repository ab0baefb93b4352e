// What the decodes over caches of few bits share: all slices' keys, in steps of kTile, are one sequence that is cut into equal parts, one for each warp on the
// GPU whatever the lengths are.  A slice (batch entry, key/value head, tile of its query heads) that one warp has to itself is written at once; of others
// each warp leaves a normalised result and its log-sum-exp, which a second kernel merges.
#pragma once
#include "common.h"

namespace ttk {

// m16n8k16 in halves with 32-bit sums, and with sums that begin here
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

struct PartsArgs {
    const __nv_bfloat16* q;
    const unsigned char *kc, *vc;
    const int *table, *lens;
    int B, L, hkv, group, head_tiles, n_pages, page, max_pages;
    float scale_log2;
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
struct PartsShares {
    unsigned parts, per, rest;
    __host__ __device__ __forceinline__ PartsShares(unsigned total, unsigned warps, unsigned slices) {
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

__device__ __forceinline__ int parts_len(const PartsArgs& a, int b) { return a.lens ? min(max(__ldg(a.lens + b), 0), a.L) : a.L; }
template <int kTile>
__device__ __forceinline__ unsigned parts_steps(int len) {
    return (unsigned)(len + kTile - 1) / kTile;
}

// A place in the sequence of steps: the batch entry it is in and where that one's steps begin.
template <int kTile>
struct PartsCursor {
    int b, len;
    unsigned begin;
    __device__ __forceinline__ void to(const PartsArgs& a, unsigned per_b, unsigned x) {   // x >= begin, below the end
        unsigned n;
        while (x - begin >= (n = parts_steps<kTile>(len) * per_b)) {
            begin += n;
            len = parts_len(a, ++b);
        }
    }
    // the slice within the batch entry, and the step within the slice
    __device__ __forceinline__ int slice(unsigned x, int* step) const {
        const unsigned steps = parts_steps<kTile>(len), s = (x - begin) / steps;
        *step = (int)(x - begin - s * steps);
        return (int)s;
    }
};

// Where warp w's part begins: its cursor, first step and number of steps; false where it has none (a sequence without keys that is one warp's gets its
// zeros here).  The whole warp calls it.
template <int kTile, int D, int kHeads>
__device__ __forceinline__ bool parts_find(const PartsArgs& a, unsigned w, unsigned w_all, int lane, PartsCursor<kTile>* now, unsigned* x0, int* n) {
    const unsigned per_b = a.hkv * a.head_tiles;
    if (!a.before) {   // a slice to a warp
        if (w >= a.B * per_b) return false;
        now->b = w / per_b;
        now->len = parts_len(a, now->b);
        *n = (int)parts_steps<kTile>(now->len);
        *x0 = (w - now->b * per_b) * *n;   // (with the batch entry's own first step as 0)
        if (*n == 0) {
            const int slice_b = w - now->b * per_b, h0 = slice_b % a.head_tiles * kHeads, n_heads = min(kHeads, a.group - h0);
            const long long row0 = ((long long)now->b * a.hkv + slice_b / a.head_tiles) * a.group + h0;
            for (int i = lane; i < n_heads * (D / 8); i += 32) reinterpret_cast<uint4*>(a.out + row0 * D)[i] = make_uint4(0, 0, 0, 0);
            if (lane < n_heads && a.lse) a.lse[row0 + lane] = -INFINITY;
            return false;
        }
    } else {
        // the batch's steps, and where this warp's part begins
        unsigned sum = 0;
        for (int i = lane; i < a.B; i += 32) sum += parts_steps<kTile>(parts_len(a, i));
        const unsigned total = __reduce_add_sync(0xffffffffu, sum) * per_b;
        const PartsShares shares(total, w_all, a.B * per_b);
        if (w >= shares.parts) return false;
        *x0 = shares.begin(w);
        *n = (int)(shares.begin(w + 1) - *x0);
        const unsigned y = *x0 / per_b;
        unsigned done = 0;
        int found = -1;
        for (int i = 0; i < a.B && (found < 0 || w == 0); i += 32) {
            const int len = i + lane < a.B ? parts_len(a, i + lane) : 0;
            unsigned to = parts_steps<kTile>(len);
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
                now->b = found;
                now->len = __shfl_sync(0xffffffffu, len, at);
                now->begin = (__shfl_sync(0xffffffffu, to, at) - parts_steps<kTile>(now->len)) * per_b;
            }
            done = __shfl_sync(0xffffffffu, to, 31);
        }
        if (found < 0) return false;   // no keys at all
    }
    return true;
}

// The merge of the parts that n_warps warps have left (attn_decode_q4.cu).
template <int D>
cudaError_t decode_parts_merge(const PartsArgs& g, const AttnArgs& a, int n_warps, cudaStream_t st);

}  // namespace ttk
