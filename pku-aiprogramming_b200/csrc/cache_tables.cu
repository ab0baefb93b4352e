// Page tables of a paged cache from the requests' lengths: pages and slots for new tokens, and pages given back.
//
// With c(n) = ceil(n / page): request b needs c(len + new) - c(len) pages; its first page and first packed row are exclusive sums
// over the requests before it, and whether it is served is a comparison of the inclusive sums with what there is, so the
// served requests are a prefix.  Token t of a request is at position p = len + t, in the row's column p / page.
//
// The bytes are few (4 per length, 8 per token and page), so what counts is the number of launches and of dependent loads in
// one: every CTA sums over all requests itself (a few loads per thread, from L2) instead of waiting for a launch that
// does, and a token finds its request by a binary search in shared memory.  Nothing is kept between calls.  Giving pages back
// is the work of one CTA where an entry is no page, since where a page goes depends on how many before it are.
#include <climits>

#include "common.h"

namespace ttk {

constexpr int kMaxRequests = 16384;   // three ints each in shared memory
int cache_max_requests() { return kMaxRequests; }

// Inclusive sums over the CTA's threads; `red` [2][32] shared, used once per kernel.
template <int kThreads>
__device__ __forceinline__ void cta_sums(long long& a, long long& b, long long (*red)[32]) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) {
            a += x;
            b += y;
        }
    }
    if (lane == 31) {
        red[0][w] = a;
        red[1][w] = b;
    }
    __syncthreads();
    for (int i = 0; i < w; ++i) {
        a += red[0][i];
        b += red[1][i];
    }
}

struct Need {
    int tokens, pages, have;   // new tokens, pages to take, columns in use before
};
__device__ __forceinline__ Need need_of(int len, int fresh, int page, long long row_tokens) {
    Need n{0, 0, 0};
    if (len < 0 || fresh < 0 || (long long)len + fresh > row_tokens) return n;
    n.have = len / page + (len % page != 0);
    n.tokens = fresh;
    n.pages = (len + fresh) / page + ((len + fresh) % page != 0) - n.have;
    return n;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) cache_extend_kernel(int* __restrict__ table, const int* __restrict__ lens, const int* __restrict__ fresh,
                                                                const int* __restrict__ free_pages, const int* __restrict__ n_free, int B,
                                                                int page, int max_pages, int free_capacity, int max_tokens, int* __restrict__ lens_out,
                                                                int* __restrict__ n_free_out, int* __restrict__ cu_new, int* __restrict__ slots,
                                                                int* __restrict__ positions) {
    extern __shared__ int sm[];
    int* cu = sm;              // [B + 1] packed rows of the requests served
    int* first = sm + B + 1;   // [B] pages taken by the requests before; -1: not served
    int* held = first + B;     // [B] lens
    __shared__ long long red[2][32];
    __shared__ int total[2];
    const int tid = threadIdx.x, per = (B + kThreads - 1) / kThreads, b0 = min(B, tid * per), b1 = min(B, b0 + per);
    const long long row_tokens = min((long long)max_pages * page, (long long)INT_MAX);
    if (tid < 2) total[tid] = 0;
    grid_let_next_start();
    grid_wait_for_previous();
    const int have_free = min(max(*n_free, 0), free_capacity);
    long long tok = 0, pg = 0;
    for (int b = b0; b < b1; ++b) {
        held[b] = lens[b];
        const Need n = need_of(held[b], fresh[b], page, row_tokens);
        tok += n.tokens;
        pg += n.pages;
    }
    const long long own_tok = tok, own_pg = pg;
    cta_sums<kThreads>(tok, pg, red);   // (its barrier is behind the clearing of `total`)
    tok -= own_tok;
    pg -= own_pg;
    int most_tok = 0, most_pg = 0;
    for (int b = b0; b < b1; ++b) {
        const Need n = need_of(held[b], fresh[b], page, row_tokens);
        tok += n.tokens;
        pg += n.pages;
        const bool ok = tok <= max_tokens && pg <= have_free;
        cu[b + 1] = ok ? (int)tok : -1;
        first[b] = ok ? (int)(pg - n.pages) : -1;
        if (ok) {
            most_tok = (int)tok;
            most_pg = (int)pg;
        }
    }
    atomicMax(&total[0], most_tok);
    atomicMax(&total[1], most_pg);
    if (tid == 0) cu[0] = 0;
    __syncthreads();
    const int served = total[0];
    for (int b = b0; b < b1; ++b)
        if (cu[b + 1] < 0) cu[b + 1] = served;
    __syncthreads();
    auto from_free = [&](int i) { return free_pages[have_free - 1 - i]; };   // the i-th page taken
    if (blockIdx.x == 0) {
        for (int b = tid; b < B; b += kThreads) {
            lens_out[b] = held[b] + (cu[b + 1] - cu[b]);
            cu_new[b + 1] = cu[b + 1];
        }
        if (tid == 0) {
            cu_new[0] = 0;
            *n_free_out = have_free - total[1];
        }
    }
    // new columns: a warp per request
    for (int b = blockIdx.x * (kThreads / 32) + (tid >> 5); b < B; b += gridDim.x * (kThreads / 32)) {
        if (first[b] < 0 || cu[b + 1] == cu[b]) continue;
        const Need n = need_of(held[b], cu[b + 1] - cu[b], page, row_tokens);
        for (int j = tid & 31; j < n.pages; j += 32) table[(long long)b * max_pages + n.have + j] = from_free(first[b] + j);
    }
    for (long long t = (long long)blockIdx.x * kThreads + tid; t < max_tokens; t += (long long)gridDim.x * kThreads) {
        int slot = -1, pos = 0;
        if (t < served) {
            int lo = 0, hi = B;   // the last b with cu[b] <= t, behind requests without tokens
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int len = held[lo], have = len / page + (len % page != 0);
            pos = len + (int)(t - cu[lo]);
            const int col = pos / page;
            const int p = col < have ? table[(long long)lo * max_pages + col] : from_free(first[lo] + col - have);
            if (p >= 0) slot = p * page + (pos - col * page);
        }
        slots[t] = slot;
        positions[t] = pos;
    }
}

// Pages given back.  Entries of done requests that are no pages (negative) are left out, so a page's place behind *n_free is the number of pages among all
// entries before it.  Two kernels where there may be many: the first copies all entries to where they belong if there are no such holes, and leaves kHoles in
// the last of lens_out if it meets one; the second then does all of it anew, or else writes that length.  (What lens_out held before cannot mislead it: with
// kHoles there it does the work in vain.)
constexpr int kHoles = INT_MIN;
constexpr int kCopied = 128;
template <int kThreads>
__global__ void __launch_bounds__(kThreads) cache_copy_kernel(const int* __restrict__ table, const int* __restrict__ lens, const unsigned char* __restrict__ done,
                                                              int* __restrict__ free_pages, const int* __restrict__ n_free, int B, int page, int max_pages,
                                                              int free_capacity, int* __restrict__ lens_out, int* __restrict__ n_free_out) {
    extern __shared__ int sm[];
    int* first = sm;      // [B] where the request's pages go, behind *n_free
    int* count = sm + B;   // [B] how many there are
    __shared__ long long red[2][32];
    const int tid = threadIdx.x, per = (B + kThreads - 1) / kThreads, b0 = min(B, tid * per), b1 = min(B, b0 + per);
    grid_let_next_start();
    grid_wait_for_previous();
    const int have_free = min(max(*n_free, 0), free_capacity);
    long long pg = 0, zero = 0;
    for (int b = b0; b < b1; ++b) {
        const int len = done[b] ? lens[b] : 0;
        count[b] = len <= 0 ? 0 : min(max_pages, len / page + (len % page != 0));
        pg += count[b];
    }
    const long long own = pg;
    cta_sums<kThreads>(pg, zero, red);
    if (blockIdx.x == 0 && tid == kThreads - 1) *n_free_out = (int)min(have_free + pg, (long long)free_capacity);
    pg -= own;
    for (int b = b0; b < b1; ++b) {
        first[b] = (int)min(pg, (long long)INT_MAX);
        pg += count[b];
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = tid; b < B - 1; b += kThreads) lens_out[b] = done[b] ? 0 : lens[b];
    // a warp per kCopied columns of a request, all loads of a lane before its stores
    const unsigned pieces = (max_pages - 1) / kCopied + 1;
    for (long long item = blockIdx.x * (kThreads / 32) + (tid >> 5); item < (long long)B * pieces; item += gridDim.x * (kThreads / 32)) {
        const int b = (int)(item / pieces), j0 = (int)(item - (long long)b * pieces) * kCopied, n = count[b];
        if (j0 >= n) continue;
        int x[kCopied / 32];
        bool hole = false;
#pragma unroll
        for (int i = 0; i < kCopied / 32; ++i) {
            const int j = j0 + 32 * i + (tid & 31);
            if (j < n) x[i] = table[(long long)b * max_pages + j];
        }
#pragma unroll
        for (int i = 0; i < kCopied / 32; ++i) {
            const int j = j0 + 32 * i + (tid & 31);
            const long long to = (long long)have_free + first[b] + j;
            if (j < n && to < free_capacity) free_pages[to] = x[i];
            hole = hole || (j < n && x[i] < 0);
        }
        if (hole) lens_out[B - 1] = kHoles;
    }
}

// One CTA.  Columns in use are cut into pieces of `width`, `pieces` to a row; a warp counts the pages of a piece, all sum over all pieces, and the warp writes its
// piece's pages, which it still holds where it has one piece of kPiece entries, and else finds in the SM's cache.
constexpr int kGiveThreads = 1024, kLoads = 16, kPiece = 32 * kLoads, kMaxPieces = 2 * kMaxRequests;
__global__ void __launch_bounds__(kGiveThreads) cache_release_kernel(const int* __restrict__ table, const int* __restrict__ lens, const unsigned char* __restrict__ done,
                                                                     int* __restrict__ free_pages, const int* __restrict__ n_free, int B, int page, int max_pages,
                                                                     int free_capacity, int width, int pieces, bool copied, int* lens_out, int* __restrict__ n_free_out) {
    extern __shared__ int sm[];
    int* count = sm;      // [B] columns in use
    int* first = sm + B;   // [B * pieces] pages of a piece, and then of those before it
    __shared__ long long red[2][32];
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, items = B * pieces;
    grid_let_next_start();
    grid_wait_for_previous();
    if (copied && !__syncthreads_or(tid == 0 && lens_out[B - 1] == kHoles)) {
        if (tid == 0) lens_out[B - 1] = done[B - 1] ? 0 : lens[B - 1];
        return;
    }
    const int have_free = min(max(*n_free, 0), free_capacity);
    for (int b = tid; b < B; b += threads) {
        const int held = lens[b], len = done[b] ? held : 0;
        count[b] = len <= 0 ? 0 : min(max_pages, len / page + (len % page != 0));
    }
    __syncthreads();
    int x[kLoads];
    auto load = [&](const int* from, int n) {   // kPiece entries, of which n are there
#pragma unroll
        for (int i = 0; i < kLoads; ++i) x[i] = 32 * i + lane < n ? from[32 * i + lane] : -1;
    };
    auto piece = [&](int item, const int** from) {   // its number of entries, and the first
        const int b = item / pieces, j0 = (item - b * pieces) * width;
        *from = table + (long long)b * max_pages + j0;
        return min(count[b] - j0, width);
    };
    for (int item = tid >> 5; item < items; item += threads / 32) {
        const int* from;
        const int n = piece(item, &from);
        int here = 0;
        for (int j0 = 0; j0 < n; j0 += kPiece) {
            load(from + j0, n - j0);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) here += x[i] >= 0;
        }
        here = __reduce_add_sync(0xffffffffu, here);
        if (lane == 0) first[item] = here;
    }
    __syncthreads();
    const int per = (items + threads - 1) / threads, i0 = min(items, tid * per), i1 = min(items, i0 + per);
    long long pg = 0, zero = 0;
    for (int i = i0; i < i1; ++i) pg += first[i];
    const long long own = pg;
    cta_sums<kGiveThreads>(pg, zero, red);
    if (tid == threads - 1) *n_free_out = (int)min(have_free + pg, (long long)free_capacity);
    for (int b = tid; b < B; b += threads) {
        const int held = lens[b];
        lens_out[b] = done[b] ? 0 : held;
    }
    pg -= own;
    for (int i = i0; i < i1; ++i) {
        const int n = first[i];
        first[i] = (int)min(pg, (long long)INT_MAX);
        pg += n;
    }
    __syncthreads();
    const bool held = items <= threads / 32 && width == kPiece;
    for (int item = tid >> 5; item < items; item += threads / 32) {
        const int* from;
        const int n = piece(item, &from);
        long long to = (long long)have_free + first[item];
        for (int j0 = 0; j0 < n; j0 += kPiece) {
            if (!held) load(from + j0, n - j0);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const unsigned there = __ballot_sync(0xffffffffu, x[i] >= 0);
                const long long at = to + __popc(there & ((1u << lane) - 1));
                if (x[i] >= 0 && at < free_capacity) free_pages[at] = x[i];
                to += __popc(there);
            }
        }
    }
}

// Threads: one request each up to 256, four each beyond.  CTAs: every one sums over all requests, so not more than three to an SM (270,000 tokens of 256
// requests: 6.5 / 5.7 / 8.1 us at two, three and four).
cudaError_t cache_extend(int* table, const int* lens, const int* fresh, const int* free_pages, const int* n_free, int B, int page, int max_pages,
                         int free_capacity, int max_tokens, int* lens_out, int* n_free_out, int* cu_new, int* slots, int* positions, cudaStream_t st) {
    const size_t smem = (3 * (size_t)B + 1) * sizeof(int);
    auto go = [&](auto kernel, int threads) {
        if (smem > 48 * 1024 - 1024) {
            const cudaError_t e = TT_ALLOW_SMEM(kernel, (3 * (size_t)kMaxRequests + 1) * sizeof(int));
            if (e != cudaSuccess) return e;
        }
        const long long rows = (max_tokens + (long long)threads - 1) / threads, reqs = (B + threads / 32 - 1) / (threads / 32);
        const long long ctas = rows > reqs ? rows : reqs, most = (threads == 256 ? 3LL : 1LL) * sm_count();
        LaunchScope ls(K_CACHE_TABLES, st);
        return launch_overlapped(kernel, (unsigned)(ctas < most ? ctas : most), threads, smem, st, table, lens, fresh, free_pages, n_free, B, page,
                                 max_pages, free_capacity, max_tokens, lens_out, n_free_out, cu_new, slots, positions);
    };
    return B <= 1024 ? go(cache_extend_kernel<256>, 256) : go(cache_extend_kernel<1024>, 1024);
}
// Pages given back, us from a graph / as calls: 4 requests 3.1 / 5.0 by the one kernel, 3.3 / 7.8 by both; one with 8192 columns 4.6 / 5.0 and 3.4 / 7.4.  By both: 64 of
// up to 256 pages 3.7 / 7.1, 512 of up to 512 of which half are done, 65,000 pages, 4.6 / 7.0 (copying with a warp per request for one per 128 columns takes 2.3 more);
// all 260,000 of them 4.7 / 7.2.  With a hole the 65,000 take 33 us, those of 26 requests 18: one SM does it then, since CTAs that count together would wait for
// each other in every call to learn whether there is one (0.8 us).
cudaError_t cache_release(const int* table, const int* lens, const unsigned char* done, int* free_pages, const int* n_free, int B, int page, int max_pages,
                          int free_capacity, int* lens_out, int* n_free_out, cudaStream_t st) {
    int width = kPiece, pieces;
    while ((long long)B * (pieces = (max_pages - 1) / width + 1) > kMaxPieces) width *= 2;
    const bool copied = B * pieces > kGiveThreads / 32;
    if (copied) {
        const size_t smem = 2 * (size_t)B * sizeof(int);
        auto go = [&](auto kernel, int threads) {
            if (smem > 48 * 1024 - 1024) {
                const cudaError_t e = TT_ALLOW_SMEM(kernel, 2 * (size_t)kMaxRequests * sizeof(int));
                if (e != cudaSuccess) return e;
            }
            const long long warps = B * ((max_pages - 1LL) / kCopied + 1), ctas = (warps + threads / 32 - 1) / (threads / 32), most = (threads == 256 ? 8LL : 1LL) * sm_count();
            LaunchScope ls(K_CACHE_TABLES, st);
            return launch_overlapped(kernel, (unsigned)(ctas < most ? ctas : most), threads, smem, st, table, lens, done, free_pages, n_free, B, page, max_pages, free_capacity,
                                     lens_out, n_free_out);
        };
        const cudaError_t e = B <= 1024 ? go(cache_copy_kernel<256>, 256) : go(cache_copy_kernel<1024>, 1024);
        if (e != cudaSuccess) return e;
    }
    const size_t smem = (size_t)B * (1 + pieces) * sizeof(int);
    if (smem > 48 * 1024 - 1024) {
        const cudaError_t e = TT_ALLOW_SMEM(cache_release_kernel, (kMaxRequests + (size_t)kMaxPieces) * sizeof(int));
        if (e != cudaSuccess) return e;
    }
    LaunchScope ls(K_CACHE_TABLES, st);
    return launch_overlapped(cache_release_kernel, 1, B * pieces <= 8 ? 256 : kGiveThreads, smem, st, table, lens, done, free_pages, n_free, B, page, max_pages, free_capacity,
                             width, pieces, copied, lens_out, n_free_out);
}

}  // namespace ttk
