// C-ABI layer of what stands around a paged cache: page tables, the 4-bit cache, rotary positions.  Argument checks and launches;
// see include/tt_attn.h.
#include "../../include/tt_attn.h"
#include "common.h"

#include <cmath>
#include <cstdlib>

namespace ttk {
int resolve(const tt_attn_desc* d, AttnArgs* a, const char* who);   // tt_api.cu
namespace {

struct Span {
    const void* p;
    size_t bytes;
    const char* name;
};
bool overlap(const Span& a, const Span& b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.p && b.p && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
}
// Outputs that lie on an input or on each other: some CTAs would read what others have written.
int check_overlap(const char* who, const Span* out, int n_out, const Span* in, int n_in) {
    for (int i = 0; i < n_out; ++i) {
        for (int j = 0; j < n_in; ++j)
            if (overlap(out[i], in[j])) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].name, in[j].name);
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].name, out[j].name);
    }
    return TT_OK;
}

int table_args(const char* who, int32_t B, int32_t page_size, int32_t max_pages, int32_t free_capacity) {
    if (B < 1 || page_size < 1 || max_pages < 1 || free_capacity < 0)
        return fail(TT_ERR_BAD_SHAPE, "%s: B=%d page_size=%d max_pages=%d must be >= 1, free_capacity=%d >= 0", who, B, page_size, max_pages, free_capacity);
    if (B > cache_max_requests()) return fail(TT_ERR_BAD_SHAPE, "%s: B=%d, at most %d requests", who, B, cache_max_requests());
    return TT_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int q4_args(const char* who, const void* k_cache, const void* v_cache, int32_t Hkv, int32_t D, int32_t n_pages, int32_t page_size) {
    if (D != 64 && D != 128) return fail(TT_ERR_UNSUPPORTED, "%s: head dim 64 or 128 only, got %d", who, D);
    if (page_size < 16 || page_size % 16) return fail(TT_ERR_BAD_SHAPE, "%s: page_size=%d must be a multiple of 16", who, page_size);
    if (Hkv < 1 || n_pages < 0) return fail(TT_ERR_BAD_SHAPE, "%s: Hkv=%d n_pages=%d", who, Hkv, n_pages);
    if ((int64_t)n_pages * page_size >= (1LL << 31)) return fail(TT_ERR_BAD_SHAPE, "%s: pages of %d x %d tokens, at most 2^31 - 1", who, n_pages, page_size);
    if ((double)n_pages * Hkv * page_size * (D / 2 + D / 32) >= 137438953472.0) return fail(TT_ERR_BAD_SHAPE, "%s: a cache of 2^37 bytes or more", who);
    if (n_pages && (!k_cache || !v_cache)) return fail(TT_ERR_NULL, "%s: null cache", who);
    if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(TT_ERR_BAD_SHAPE, "%s: the cache must be 16-byte aligned", who);
    return TT_OK;
}

// Whether rows of D elements at strides st over extents n lie apart from each other.
bool rows_apart(const int64_t* st, const int* n, int D) {
    int order[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (st[order[j]] < st[order[i]]) {
                const int t = order[i];
                order[i] = order[j];
                order[j] = t;
            }
    int64_t reach = D;   // from the first element to behind the last of the dimensions so far
    for (int i = 0; i < 3; ++i) {
        const int d = order[i];
        if (n[d] == 1) continue;
        if (st[d] < reach) return false;
        reach += st[d] * (n[d] - 1);
    }
    return true;
}
// A tensor of rows of D elements at strides st over extents n, and what it spans.
struct Rows {
    const int64_t* st;
    const int* n;
    Span span;
    Rows(const void* p, const int64_t* strides, const int* extents, int D, size_t size, const char* name) : st(strides), n(extents) {
        int64_t last = D;
        for (int i = 0; i < 3; ++i) last += st[i] * (n[i] - 1);
        span = Span{p, (size_t)last * size, name};
    }
};
// Whether some row of x and some row of y share an element.  Slices of one buffer interleave without meeting: exact where x and y have the same strides
// and rows apart from each other, else by what they span.
bool rows_meet(const Rows& x, const Rows& y, int D, size_t size) {
    if (!overlap(x.span, y.span)) return false;
    int64_t st[3];
    int n[3];
    for (int i = 0; i < 3; ++i) {
        if (x.n[i] > 1 && y.n[i] > 1 && x.st[i] != y.st[i]) return true;
        st[i] = x.n[i] > 1 ? x.st[i] : y.st[i];
        n[i] = x.n[i] > y.n[i] ? x.n[i] : y.n[i];
    }
    if (!rows_apart(st, n, D)) return true;
    // rows i of x and j of y are delta + sum (i - j) st apart; from the largest stride down the rest is less than a stride, so two i - j can cancel it
    const int64_t delta = ((const char*)x.span.p - (const char*)y.span.p) / (int64_t)size;
    bool used[3] = {n[0] == 1, n[1] == 1, n[2] == 1};
    int64_t left[8] = {delta};
    int count = 1;
    for (int k = 0; k < 3; ++k) {
        int d = -1;
        for (int i = 0; i < 3; ++i)
            if (!used[i] && (d < 0 || st[i] > st[d])) d = i;
        if (d < 0) break;
        used[d] = true;
        for (int i = count - 1; i >= 0; --i) {
            const int64_t r = left[i], down = r >= 0 ? r / st[d] : -((-r + st[d] - 1) / st[d]);   // floor
            for (int e = 0; e < 2; ++e) {
                int64_t m = -down - e;   // i - j
                if (m > x.n[d] - 1) m = x.n[d] - 1;
                if (m < 1 - y.n[d]) m = 1 - y.n[d];
                left[e ? count + i : i] = r + m * st[d];
            }
        }
        count *= 2;
    }
    for (int i = 0; i < count; ++i)
        if (left[i] < D && left[i] > -D) return true;
    return false;
}

}  // namespace
}  // namespace ttk

using namespace ttk;

extern "C" {

int tt_cache_extend(int32_t* block_table, const int32_t* seq_lens, const int32_t* new_lens, const int32_t* free_pages, const int32_t* n_free, int32_t B,
                    int32_t page_size, int32_t max_pages, int32_t free_capacity, int32_t max_tokens, int32_t* seq_lens_out, int32_t* n_free_out,
                    int32_t* cu_new, int32_t* slots, int32_t* positions, void* stream) {
    const char* who = "tt_cache_extend";
    int rc = table_args(who, B, page_size, max_pages, free_capacity);
    if (rc != TT_OK) return rc;
    if (max_tokens < 0) return fail(TT_ERR_BAD_SHAPE, "%s: max_tokens=%d", who, max_tokens);
    if (!block_table || !seq_lens || !new_lens || !n_free || !seq_lens_out || !n_free_out || !cu_new || (free_capacity && !free_pages) ||
        (max_tokens && (!slots || !positions)))
        return fail(TT_ERR_NULL, "%s: null pointer", who);
    const size_t n = (size_t)B * 4, t = (size_t)max_tokens * 4;
    const Span out[] = {{seq_lens_out, n, "seq_lens_out"}, {n_free_out, 4, "n_free_out"}, {cu_new, n + 4, "cu_new"}, {slots, t, "slots"},
                        {positions, t, "positions"}, {block_table, n * max_pages, "block_table"}};
    const Span in[] = {{seq_lens, n, "seq_lens"}, {new_lens, n, "new_lens"}, {free_pages, (size_t)free_capacity * 4, "free_pages"}, {n_free, 4, "n_free"}};
    if ((rc = check_overlap(who, out, 6, in, 4)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    const cudaError_t e = cache_extend(block_table, seq_lens, new_lens, free_pages, n_free, B, page_size, max_pages, free_capacity, max_tokens, seq_lens_out,
                                       n_free_out, cu_new, slots, positions, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_cache_extend: launch");
}

int tt_cache_release(const int32_t* block_table, const int32_t* seq_lens, const uint8_t* done, int32_t* free_pages, const int32_t* n_free, int32_t B,
                     int32_t page_size, int32_t max_pages, int32_t free_capacity, int32_t* seq_lens_out, int32_t* n_free_out, void* stream) {
    const char* who = "tt_cache_release";
    int rc = table_args(who, B, page_size, max_pages, free_capacity);
    if (rc != TT_OK) return rc;
    if (!block_table || !seq_lens || !done || !n_free || !seq_lens_out || !n_free_out || (free_capacity && !free_pages))
        return fail(TT_ERR_NULL, "%s: null pointer", who);
    const size_t n = (size_t)B * 4;
    const Span out[] = {{seq_lens_out, n, "seq_lens_out"}, {n_free_out, 4, "n_free_out"}, {free_pages, (size_t)free_capacity * 4, "free_pages"}};
    const Span in[] = {{block_table, n * max_pages, "block_table"}, {seq_lens, n, "seq_lens"}, {done, (size_t)B, "done"}, {n_free, 4, "n_free"}};
    if ((rc = check_overlap(who, out, 3, in, 4)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    const cudaError_t e = cache_release(block_table, seq_lens, done, free_pages, n_free, B, page_size, max_pages, free_capacity, seq_lens_out, n_free_out,
                                        (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_cache_release: launch");
}

size_t tt_cache_q4_page_bytes(int32_t page_size, int32_t D) {
    if ((D != 64 && D != 128) || page_size < 16 || page_size % 16) return 0;
    return (size_t)page_size * (D / 2 + D / 32);
}

int tt_cache_append_q4(const void* k, const void* v, const int32_t* slots, int32_t T, int32_t Hkv, int32_t D, int32_t dtype, const int64_t* k_stride,
                       const int64_t* v_stride, void* k_cache, void* v_cache, int32_t n_pages, int32_t page_size, void* stream) {
    const char* who = "tt_cache_append_q4";
    int rc = q4_args(who, k_cache, v_cache, Hkv, D, n_pages, page_size);
    if (rc != TT_OK) return rc;
    if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_BAD_DTYPE, "%s: dtype %d unknown", who, dtype);
    if (T < 0 || (int64_t)T * Hkv >= (1LL << 31)) return fail(TT_ERR_BAD_SHAPE, "%s: T=%d Hkv=%d", who, T, Hkv);
    if (!k_stride || !v_stride) return fail(TT_ERR_NULL, "%s: null strides", who);
    if (T && (!k || !v || !slots)) return fail(TT_ERR_NULL, "%s: null pointer", who);
    const size_t size = dtype == TT_BF16 ? 2 : 4;
    if (((uintptr_t)k | (uintptr_t)v) % size) return fail(TT_ERR_BAD_SHAPE, "%s: pointers must be multiples of the element size", who);
    if (k_stride[0] < 0 || k_stride[1] < 0 || v_stride[0] < 0 || v_stride[1] < 0) return fail(TT_ERR_BAD_SHAPE, "%s: negative stride", who);
    const size_t pool = (size_t)n_pages * Hkv * tt_cache_q4_page_bytes(page_size, D);
    auto bytes = [&](const int64_t* st) { return T ? (size_t)((T - 1) * st[0] + (Hkv - 1) * st[1] + D) * size : 0; };
    const Span out[] = {{k_cache, pool, "k_cache"}, {v_cache, pool, "v_cache"}}, in[] = {{k, bytes(k_stride), "k"}, {v, bytes(v_stride), "v"}, {slots, (size_t)T * 4, "slots"}};
    if ((rc = check_overlap(who, out, 2, in, 3)) != TT_OK) return rc;
    if ((rc = check_device()) != TT_OK || T == 0 || n_pages == 0) return rc;
    const CacheQ4 c{k_cache, v_cache, n_pages, page_size, Hkv, D};
    const long long ks[2] = {k_stride[0], k_stride[1]}, vs[2] = {v_stride[0], v_stride[1]};
    const cudaError_t e = cache_append_q4(c, k, v, ks, vs, dtype == TT_BF16, slots, T, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_cache_append_q4: launch");
}

int tt_cache_read_q4(const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* cu_lens, int32_t B, int32_t Hkv, int32_t D,
                     int32_t n_pages, int32_t page_size, int32_t max_pages, int32_t total, void* k, void* v, void* stream) {
    const char* who = "tt_cache_read_q4";
    int rc = q4_args(who, k_cache, v_cache, Hkv, D, n_pages, page_size);
    if (rc != TT_OK) return rc;
    if (B < 1 || max_pages < 1 || total < 0 || (int64_t)total * Hkv >= (1LL << 31))
        return fail(TT_ERR_BAD_SHAPE, "%s: B=%d max_pages=%d total=%d Hkv=%d", who, B, max_pages, total, Hkv);
    if (!block_table || !cu_lens || (total && (!k || !v))) return fail(TT_ERR_NULL, "%s: null pointer", who);
    if (!aligned16(k) || !aligned16(v)) return fail(TT_ERR_BAD_SHAPE, "%s: k and v must be 16-byte aligned", who);
    const size_t pool = (size_t)n_pages * Hkv * tt_cache_q4_page_bytes(page_size, D), n = (size_t)total * Hkv * D * 2;
    const Span out[] = {{k, n, "k"}, {v, n, "v"}};
    const Span in[] = {{k_cache, pool, "k_cache"}, {v_cache, pool, "v_cache"}, {block_table, (size_t)B * max_pages * 4, "block_table"}, {cu_lens, ((size_t)B + 1) * 4, "cu_lens"}};
    if ((rc = check_overlap(who, out, 2, in, 4)) != TT_OK || (rc = check_device()) != TT_OK || total == 0) return rc;
    const CacheQ4 c{const_cast<void*>(k_cache), const_cast<void*>(v_cache), n_pages, page_size, Hkv, D};
    const cudaError_t e = cache_read_q4(c, block_table, cu_lens, B, max_pages, total, k, v, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_cache_read_q4: launch");
}

static int resolve_q4(const char* who, const tt_attn_desc* desc, AttnArgs* a) {
    const int rc = resolve(desc, a, who);
    if (rc != TT_OK) return rc;
    if (a->S != 1) return fail(TT_ERR_BAD_SHAPE, "%s: S must be 1, got %d", who, a->S);
    if (!a->bf16 || (a->D != 64 && a->D != 128)) return fail(TT_ERR_BAD_DTYPE, "%s: bf16 with D = 64 or 128 only (dtype %d, D %d)", who, desc->dtype, a->D);
    if (a->L > (1 << 30)) return fail(TT_ERR_BAD_SHAPE, "%s: L=%d exceeds 2^30", who, a->L);
    a->causal = 0;
    return TT_OK;
}
size_t tt_attn_decode_q4_workspace_bytes(const tt_attn_desc* desc) {
    AttnArgs a;
    return resolve_q4("tt_attn_decode_q4_workspace_bytes", desc, &a) == TT_OK ? attn_decode_q4_workspace(a) : 0;
}
int tt_attn_decode_q4(const tt_attn_desc* desc, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* seq_lens,
                      int32_t n_pages, int32_t page_size, int32_t max_pages, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "tt_attn_decode_q4";
    AttnArgs a;
    int rc = resolve_q4(who, desc, &a);
    if (rc != TT_OK) return rc;
    const int hkv = desc->H / a.group;
    if ((rc = q4_args(who, k_cache, v_cache, hkv, a.D, n_pages, page_size)) != TT_OK) return rc;
    if (!q || !out) return fail(TT_ERR_NULL, "%s: q and out must be non-null", who);
    if (!aligned16(q) || !aligned16(out)) return fail(TT_ERR_BAD_SHAPE, "%s: q and out must be 16-byte aligned", who);
    if (block_table) {
        if (max_pages < 1 || (int64_t)page_size * max_pages < a.L)
            return fail(TT_ERR_BAD_SHAPE, "%s: L=%d exceeds page_size*max_pages=%lld", who, a.L, (long long)page_size * max_pages);
    } else if (page_size < a.L || n_pages < desc->B) {
        return fail(TT_ERR_BAD_SHAPE, "%s: without a block table page_size=%d must hold L=%d and n_pages=%d the batch of %d", who, page_size, a.L, n_pages, desc->B);
    }
    const size_t need = attn_decode_q4_workspace(a);
    if (need && (!workspace || workspace_bytes < need)) return fail(TT_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, workspace_bytes);
    if (need && ((uintptr_t)workspace & 255)) return fail(TT_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    const size_t rows = (size_t)a.BH * a.D * 2, pool = (size_t)n_pages * hkv * tt_cache_q4_page_bytes(page_size, a.D);
    const Span outs[] = {{out, rows, "out"}, {lse, (size_t)a.BH * 4, "lse"}, {workspace, need, "workspace"}};
    const Span ins[] = {{q, rows, "q"}, {k_cache, pool, "k_cache"}, {v_cache, pool, "v_cache"}, {seq_lens, (size_t)desc->B * 4, "seq_lens"},
                        {block_table, block_table ? (size_t)desc->B * max_pages * 4 : 0, "block_table"}};
    if ((rc = check_overlap(who, outs, 3, ins, 5)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    a.q = q; a.out = out; a.lse = lse;
    const CacheQ4 c{const_cast<void*>(k_cache), const_cast<void*>(v_cache), n_pages, page_size, hkv, a.D};
    const cudaError_t e = attn_decode_q4(a, c, block_table, seq_lens, max_pages, workspace, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_attn_decode_q4: launch");
}

int tt_rotary(const tt_rotary_desc* d, const void* q, const void* k, const int32_t* positions, const double* inv_freq, const int32_t* axes, int32_t backward,
              void* q_out, void* k_out, void* stream) {
    const char* who = "tt_rotary";
    if (!d) return fail(TT_ERR_NULL, "%s: desc is null", who);
    const int hk = k ? d->Hkv : 0;
    if (d->B < 0 || d->S < 0 || d->H < 1 || (k && hk < 1)) return fail(TT_ERR_BAD_SHAPE, "%s: B=%d S=%d H=%d Hkv=%d", who, d->B, d->S, d->H, d->Hkv);
    if (d->D < 2 || d->D > 256 || d->R < 2 || d->R > d->D || d->R % 2)
        return fail(TT_ERR_BAD_SHAPE, "%s: D=%d must be 2..256 and R=%d even, 2..D", who, d->D, d->R);
    if (d->n_axes < 1) return fail(TT_ERR_BAD_SHAPE, "%s: n_axes=%d", who, d->n_axes);
    if (d->dtype != TT_F32 && d->dtype != TT_BF16) return fail(TT_ERR_BAD_DTYPE, "%s: dtype %d unknown", who, d->dtype);
    if (!std::isfinite(d->scale)) return fail(TT_ERR_BAD_SHAPE, "%s: scale is not finite", who);
    if ((int64_t)d->B * d->S >= (1LL << 31) || (int64_t)d->H + hk >= (1LL << 24)) return fail(TT_ERR_BAD_SHAPE, "%s: more than 2^31-1 tokens or 2^24 heads", who);
    if ((k == nullptr) != (k_out == nullptr)) return fail(TT_ERR_NULL, "%s: k and k_out go together", who);
    if (d->B == 0 || d->S == 0) return TT_OK;
    if (!q || !q_out || !positions || !inv_freq) return fail(TT_ERR_NULL, "%s: null pointer", who);
    const size_t size = d->dtype == TT_BF16 ? 2 : 4;
    const int nq[3] = {d->B, d->H, d->S}, nk[3] = {d->B, hk, d->S};
    for (int i = 0; i < 3; ++i)
        if (d->q_stride[i] < 0 || d->q_out_stride[i] < 0 || (k && (d->k_stride[i] < 0 || d->k_out_stride[i] < 0)) || (i < 2 && d->pos_stride[i] < 0))
            return fail(TT_ERR_BAD_SHAPE, "%s: negative stride", who);
    if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out) % size) return fail(TT_ERR_BAD_SHAPE, "%s: pointers must be multiples of the element size", who);
    if (!rows_apart(d->q_out_stride, nq, d->D) || (k && !rows_apart(d->k_out_stride, nk, d->D)))
        return fail(TT_ERR_BAD_SHAPE, "%s: rows of an output overlap", who);
    // An output lies on its own input row by row, or apart from everything.
    const Rows in[2] = {{q, d->q_stride, nq, d->D, size, "q"}, {k, d->k_stride, nk, d->D, size, "k"}};
    const Rows out[2] = {{q_out, d->q_out_stride, nq, d->D, size, "q_out"}, {k_out, d->k_out_stride, nk, d->D, size, "k_out"}};
    auto in_place = [](const Rows& x, const Rows& y) {
        for (int i = 0; i < 3; ++i)
            if (x.n[i] > 1 && x.st[i] != y.st[i]) return false;
        return x.span.p == y.span.p;
    };
    for (int i = 0; i < (k ? 2 : 1); ++i)
        for (int j = 0; j < (k ? 2 : 1); ++j)
            if (!(i == j && in_place(out[i], in[j])) && rows_meet(out[i], in[j], d->D, size))
                return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].span.name, in[j].span.name);
    if (k && rows_meet(out[0], out[1], d->D, size)) return fail(TT_ERR_BAD_SHAPE, "%s: q_out overlaps k_out", who);
    const size_t n_pos = (size_t)((d->n_axes - 1) * d->pos_stride[0] + (d->B - 1) * d->pos_stride[1] + d->S);
    const Span angles[] = {{positions, n_pos * 4, "positions"}, {inv_freq, (size_t)d->R / 2 * 8, "inv_freq"}, {axes, (size_t)d->R / 2 * 4, "axes"}};
    for (int i = 0; i < (k ? 2 : 1); ++i)
        for (const Span& in : angles)
            if (overlap(out[i].span, in)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].span.name, in.name);
    const int rc = check_device();
    if (rc != TT_OK) return rc;
    RotaryArgs a = {};
    a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out;
    for (int i = 0; i < 3; ++i) {
        a.xs[0][i] = d->q_stride[i]; a.xs[1][i] = d->k_stride[i];
        a.ys[0][i] = d->q_out_stride[i]; a.ys[1][i] = d->k_out_stride[i];
    }
    a.heads[0] = d->H; a.heads[1] = hk;
    a.B = d->B; a.S = d->S; a.D = d->D; a.R = d->R; a.n_axes = d->n_axes;
    a.pos = positions; a.pos_axis = d->pos_stride[0]; a.pos_batch = d->pos_stride[1];
    a.inv_freq = inv_freq; a.axes = axes; a.scale = d->scale; a.back = backward != 0;
    const cudaError_t e = rotary(a, d->dtype == TT_BF16, d->interleaved != 0, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_rotary: launch");
}

}  // extern "C"
