// C-ABI layer of what stands around a paged cache: page tables, the 4-bit cache, rotary positions.  Argument checks and launches;
// see include/tt_attn.h.
#include "../../include/tt_attn.h"
#include "common.h"

#include <cmath>
#include <cstdio>
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
// page_bytes: of one head's page, 0 where the size is not supported
int cache_args(const char* who, const void* k_cache, const void* v_cache, int32_t Hkv, int32_t D, int32_t n_pages, int32_t page_size, size_t page_bytes) {
    if (D != 64 && D != 128) return fail(TT_ERR_UNSUPPORTED, "%s: head dim 64 or 128 only, got %d", who, D);
    if (page_size < 16 || page_size % 16) return fail(TT_ERR_BAD_SHAPE, "%s: page_size=%d must be a multiple of 16", who, page_size);
    if (Hkv < 1 || n_pages < 0) return fail(TT_ERR_BAD_SHAPE, "%s: Hkv=%d n_pages=%d", who, Hkv, n_pages);
    if ((int64_t)n_pages * page_size >= (1LL << 31)) return fail(TT_ERR_BAD_SHAPE, "%s: pages of %d x %d tokens, at most 2^31 - 1", who, n_pages, page_size);
    if ((double)n_pages * Hkv * page_bytes >= 137438953472.0) return fail(TT_ERR_BAD_SHAPE, "%s: a cache of 2^37 bytes or more", who);
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

size_t element(const tt_rotary_desc* d) { return d->dtype == TT_BF16 ? 2 : 4; }
int rotary_desc_args(const char* who, const tt_rotary_desc* d, bool with_q, bool with_k) {
    if (!d) return fail(TT_ERR_NULL, "%s: desc is null", who);
    const int hk = with_k ? d->Hkv : 0;
    if (d->B < 0 || d->S < 0 || (with_q && d->H < 1) || (with_k && hk < 1)) return fail(TT_ERR_BAD_SHAPE, "%s: B=%d S=%d H=%d Hkv=%d", who, d->B, d->S, d->H, d->Hkv);
    if (d->D < 2 || d->D > 256 || d->R < 2 || d->R > d->D || d->R % 2)
        return fail(TT_ERR_BAD_SHAPE, "%s: D=%d must be 2..256 and R=%d even, 2..D", who, d->D, d->R);
    if (d->n_axes < 1) return fail(TT_ERR_BAD_SHAPE, "%s: n_axes=%d", who, d->n_axes);
    if (d->dtype != TT_F32 && d->dtype != TT_BF16) return fail(TT_ERR_BAD_DTYPE, "%s: dtype %d unknown", who, d->dtype);
    if (!std::isfinite(d->scale)) return fail(TT_ERR_BAD_SHAPE, "%s: scale is not finite", who);
    if ((int64_t)d->B * d->S >= (1LL << 31) || (int64_t)(with_q ? d->H : 0) + hk >= (1LL << 24)) return fail(TT_ERR_BAD_SHAPE, "%s: more than 2^31-1 tokens or 2^24 heads", who);
    return TT_OK;
}
int norm_args(const char* who, const tt_rotary_desc* d, int32_t weight_dtype, float eps) {
    if (weight_dtype != TT_F32 && weight_dtype != TT_BF16) return fail(TT_ERR_BAD_DTYPE, "%s: weight dtype %d unknown", who, weight_dtype);
    if (!(eps > 0.f) || !std::isfinite(eps)) return fail(TT_ERR_BAD_SHAPE, "%s: eps must be positive and finite", who);
    return TT_OK;
}
bool in_place(const Rows& x, const Rows& y) {
    for (int i = 0; i < 3; ++i)
        if (x.n[i] > 1 && x.st[i] != y.st[i]) return false;
    return x.span.p == y.span.p;
}
// Query and key heads and what becomes of them.
struct Heads {
    int n[2][3], count;
    size_t size;
    Rows in[2], out[2];
    Heads(const tt_rotary_desc* d, const void* q, const void* k, const void* q_out, const void* k_out, size_t element)
        : n{{d->B, d->H, d->S}, {d->B, k ? d->Hkv : 0, d->S}}, count(k ? 2 : 1), size(element),
          in{{q, d->q_stride, n[0], d->D, element, "q"}, {k, d->k_stride, n[1], d->D, element, "k"}},
          out{{q_out, d->q_out_stride, n[0], d->D, element, "q_out"}, {k_out, d->k_out_stride, n[1], d->D, element, "k_out"}} {}
    // An output lies on its own input row by row, or apart from everything.
    int check(const char* who, const tt_rotary_desc* d) const {
        for (int i = 0; i < 3; ++i)
            if (d->q_stride[i] < 0 || d->q_out_stride[i] < 0 || (count > 1 && (d->k_stride[i] < 0 || d->k_out_stride[i] < 0)) || (i < 2 && d->pos_stride[i] < 0))
                return fail(TT_ERR_BAD_SHAPE, "%s: negative stride", who);
        if (((uintptr_t)in[0].span.p | (uintptr_t)out[0].span.p | (uintptr_t)in[1].span.p | (uintptr_t)out[1].span.p) % size)
            return fail(TT_ERR_BAD_SHAPE, "%s: pointers must be multiples of the element size", who);
        if (!rows_apart(d->q_out_stride, n[0], d->D) || (count > 1 && !rows_apart(d->k_out_stride, n[1], d->D)))
            return fail(TT_ERR_BAD_SHAPE, "%s: rows of an output overlap", who);
        for (int i = 0; i < count; ++i)
            for (int j = 0; j < count; ++j)
                if (!(i == j && in_place(out[i], in[j])) && rows_meet(out[i], in[j], d->D, size))
                    return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].span.name, in[j].span.name);
        if (count > 1 && rows_meet(out[0], out[1], d->D, size)) return fail(TT_ERR_BAD_SHAPE, "%s: q_out overlaps k_out", who);
        return TT_OK;
    }
};
Span positions_span(const tt_rotary_desc* d, const int32_t* positions) {
    return {positions, (size_t)((d->n_axes - 1) * d->pos_stride[0] + (d->B - 1) * d->pos_stride[1] + d->S) * 4, "positions"};
}
int rotary_spans(const char* who, const Heads& h, const tt_rotary_desc* d, const int32_t* positions, const double* inv_freq, const int32_t* axes) {
    const Span angles[] = {positions_span(d, positions), {inv_freq, (size_t)d->R / 2 * 8, "inv_freq"}, {axes, (size_t)d->R / 2 * 4, "axes"}};
    for (int i = 0; i < h.count; ++i)
        for (const Span& x : angles)
            if (overlap(h.out[i].span, x)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, h.out[i].span.name, x.name);
    return TT_OK;
}
int weight_spans(const char* who, const Heads& h, const tt_rotary_desc* d, const void* q_weight, const void* k_weight, int32_t dtype) {
    const size_t size = dtype == TT_BF16 ? 2 : 4, w = (size_t)d->D * size;
    if (((uintptr_t)q_weight | (h.count > 1 ? (uintptr_t)k_weight : 0)) % size) return fail(TT_ERR_BAD_SHAPE, "%s: weights must be multiples of their element size", who);
    const Span weights[] = {{q_weight, w, "q_weight"}, {h.count > 1 ? k_weight : nullptr, w, "k_weight"}};
    for (int i = 0; i < h.count; ++i)
        for (const Span& x : weights)
            if (overlap(h.out[i].span, x)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, h.out[i].span.name, x.name);
    return TT_OK;
}
RotaryArgs rotary_args(const tt_rotary_desc* d, const void* q, const void* k, const int32_t* positions, const double* inv_freq, const int32_t* axes, void* q_out, void* k_out) {
    RotaryArgs a = {};
    a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out;
    for (int i = 0; i < 3; ++i) {
        a.xs[0][i] = d->q_stride[i]; a.xs[1][i] = d->k_stride[i];
        a.ys[0][i] = d->q_out_stride[i]; a.ys[1][i] = d->k_out_stride[i];
    }
    a.heads[0] = q ? d->H : 0; a.heads[1] = k ? d->Hkv : 0;
    a.B = d->B; a.S = d->S; a.D = d->D; a.R = d->R; a.n_axes = d->n_axes;
    a.pos = positions; a.pos_axis = d->pos_stride[0]; a.pos_batch = d->pos_stride[1];
    a.inv_freq = inv_freq; a.axes = axes; a.scale = d->scale;
    return a;
}

int launch_fail(cudaError_t e, const char* who) {
    char what[64];
    snprintf(what, sizeof what, "%s: launch", who);
    return cuda_fail(e, what);
}

// What the calls of the two caches have in common; `run` launches.
int append_to_cache(const char* who, size_t page_bytes, decltype(&cache_append_q4) run, const void* k, const void* v, const int32_t* slots, int32_t T, int32_t Hkv, int32_t D, int32_t dtype, const int64_t* k_stride,
                       const int64_t* v_stride, void* k_cache, void* v_cache, int32_t n_pages, int32_t page_size, void* stream) {
    int rc = cache_args(who, k_cache, v_cache, Hkv, D, n_pages, page_size, page_bytes);
    if (rc != TT_OK) return rc;
    if (dtype != TT_F32 && dtype != TT_BF16) return fail(TT_ERR_BAD_DTYPE, "%s: dtype %d unknown", who, dtype);
    if (T < 0 || (int64_t)T * Hkv >= (1LL << 31)) return fail(TT_ERR_BAD_SHAPE, "%s: T=%d Hkv=%d", who, T, Hkv);
    if (!k_stride || !v_stride) return fail(TT_ERR_NULL, "%s: null strides", who);
    if (T && (!k || !v || !slots)) return fail(TT_ERR_NULL, "%s: null pointer", who);
    const size_t size = dtype == TT_BF16 ? 2 : 4;
    if (((uintptr_t)k | (uintptr_t)v) % size) return fail(TT_ERR_BAD_SHAPE, "%s: pointers must be multiples of the element size", who);
    if (k_stride[0] < 0 || k_stride[1] < 0 || v_stride[0] < 0 || v_stride[1] < 0) return fail(TT_ERR_BAD_SHAPE, "%s: negative stride", who);
    const size_t pool = (size_t)n_pages * Hkv * page_bytes;
    auto bytes = [&](const int64_t* st) { return T ? (size_t)((T - 1) * st[0] + (Hkv - 1) * st[1] + D) * size : 0; };
    const Span out[] = {{k_cache, pool, "k_cache"}, {v_cache, pool, "v_cache"}}, in[] = {{k, bytes(k_stride), "k"}, {v, bytes(v_stride), "v"}, {slots, (size_t)T * 4, "slots"}};
    if ((rc = check_overlap(who, out, 2, in, 3)) != TT_OK) return rc;
    if ((rc = check_device()) != TT_OK || T == 0 || n_pages == 0) return rc;
    const CacheView c{k_cache, v_cache, n_pages, page_size, Hkv, D};
    const long long ks[2] = {k_stride[0], k_stride[1]}, vs[2] = {v_stride[0], v_stride[1]};
    const cudaError_t e = run(c, k, v, ks, vs, dtype == TT_BF16, slots, T, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : launch_fail(e, who);
}

int read_from_cache(const char* who, size_t page_bytes, decltype(&cache_read_q4) run, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* cu_lens, int32_t B, int32_t Hkv, int32_t D,
                     int32_t n_pages, int32_t page_size, int32_t max_pages, int32_t total, void* k, void* v, void* stream) {
    int rc = cache_args(who, k_cache, v_cache, Hkv, D, n_pages, page_size, page_bytes);
    if (rc != TT_OK) return rc;
    if (B < 1 || max_pages < 1 || total < 0 || (int64_t)total * Hkv >= (1LL << 31))
        return fail(TT_ERR_BAD_SHAPE, "%s: B=%d max_pages=%d total=%d Hkv=%d", who, B, max_pages, total, Hkv);
    if (!block_table || !cu_lens || (total && (!k || !v))) return fail(TT_ERR_NULL, "%s: null pointer", who);
    if (!aligned16(k) || !aligned16(v)) return fail(TT_ERR_BAD_SHAPE, "%s: k and v must be 16-byte aligned", who);
    const size_t pool = (size_t)n_pages * Hkv * page_bytes, n = (size_t)total * Hkv * D * 2;
    const Span out[] = {{k, n, "k"}, {v, n, "v"}};
    const Span in[] = {{k_cache, pool, "k_cache"}, {v_cache, pool, "v_cache"}, {block_table, (size_t)B * max_pages * 4, "block_table"}, {cu_lens, ((size_t)B + 1) * 4, "cu_lens"}};
    if ((rc = check_overlap(who, out, 2, in, 4)) != TT_OK || (rc = check_device()) != TT_OK || total == 0) return rc;
    const CacheView c{const_cast<void*>(k_cache), const_cast<void*>(v_cache), n_pages, page_size, Hkv, D};
    const cudaError_t e = run(c, block_table, cu_lens, B, max_pages, total, k, v, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : launch_fail(e, who);
}

int resolve_cache(const char* who, const tt_attn_desc* desc, AttnArgs* a) {
    const int rc = resolve(desc, a, who);
    if (rc != TT_OK) return rc;
    if (a->S != 1) return fail(TT_ERR_BAD_SHAPE, "%s: S must be 1, got %d", who, a->S);
    if (!a->bf16 || (a->D != 64 && a->D != 128)) return fail(TT_ERR_BAD_DTYPE, "%s: bf16 with D = 64 or 128 only (dtype %d, D %d)", who, desc->dtype, a->D);
    if (a->L > (1 << 30)) return fail(TT_ERR_BAD_SHAPE, "%s: L=%d exceeds 2^30", who, a->L);
    a->causal = 0;
    return TT_OK;
}
int decode_cache(const char* who, decltype(&tt_cache_q4_page_bytes) page_bytes, decltype(&attn_decode_q4_workspace) need_of, decltype(&attn_decode_q4) run, const tt_attn_desc* desc, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* seq_lens,
                      int32_t n_pages, int32_t page_size, int32_t max_pages, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    AttnArgs a;
    int rc = resolve_cache(who, desc, &a);
    if (rc != TT_OK) return rc;
    const int hkv = desc->H / a.group;
    if ((rc = cache_args(who, k_cache, v_cache, hkv, a.D, n_pages, page_size, page_bytes(page_size, a.D))) != TT_OK) return rc;
    if (!q || !out) return fail(TT_ERR_NULL, "%s: q and out must be non-null", who);
    if (!aligned16(q) || !aligned16(out)) return fail(TT_ERR_BAD_SHAPE, "%s: q and out must be 16-byte aligned", who);
    if (block_table) {
        if (max_pages < 1 || (int64_t)page_size * max_pages < a.L)
            return fail(TT_ERR_BAD_SHAPE, "%s: L=%d exceeds page_size*max_pages=%lld", who, a.L, (long long)page_size * max_pages);
    } else if (page_size < a.L || n_pages < desc->B) {
        return fail(TT_ERR_BAD_SHAPE, "%s: without a block table page_size=%d must hold L=%d and n_pages=%d the batch of %d", who, page_size, a.L, n_pages, desc->B);
    }
    const size_t need = need_of(a);
    if (need && (!workspace || workspace_bytes < need)) return fail(TT_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, workspace_bytes);
    if (need && ((uintptr_t)workspace & 255)) return fail(TT_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    const size_t rows = (size_t)a.BH * a.D * 2, pool = (size_t)n_pages * hkv * page_bytes(page_size, a.D);
    const Span outs[] = {{out, rows, "out"}, {lse, (size_t)a.BH * 4, "lse"}, {workspace, need, "workspace"}};
    const Span ins[] = {{q, rows, "q"}, {k_cache, pool, "k_cache"}, {v_cache, pool, "v_cache"}, {seq_lens, (size_t)desc->B * 4, "seq_lens"},
                        {block_table, block_table ? (size_t)desc->B * max_pages * 4 : 0, "block_table"}};
    if ((rc = check_overlap(who, outs, 3, ins, 5)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    a.q = q; a.out = out; a.lse = lse;
    const CacheView c{const_cast<void*>(k_cache), const_cast<void*>(v_cache), n_pages, page_size, hkv, a.D};
    const cudaError_t e = run(a, c, block_table, seq_lens, max_pages, workspace, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : launch_fail(e, who);
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
    return append_to_cache("tt_cache_append_q4", tt_cache_q4_page_bytes(page_size, D), cache_append_q4, k, v, slots, T, Hkv, D, dtype, k_stride, v_stride, k_cache, v_cache, n_pages, page_size, stream);
}

int tt_cache_read_q4(const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* cu_lens, int32_t B, int32_t Hkv, int32_t D,
                     int32_t n_pages, int32_t page_size, int32_t max_pages, int32_t total, void* k, void* v, void* stream) {
    return read_from_cache("tt_cache_read_q4", tt_cache_q4_page_bytes(page_size, D), cache_read_q4, k_cache, v_cache, block_table, cu_lens, B, Hkv, D, n_pages, page_size, max_pages, total, k, v, stream);
}

size_t tt_attn_decode_q4_workspace_bytes(const tt_attn_desc* desc) {
    AttnArgs a;
    return resolve_cache("tt_attn_decode_q4_workspace_bytes", desc, &a) == TT_OK ? attn_decode_q4_workspace(a) : 0;
}
int tt_attn_decode_q4(const tt_attn_desc* desc, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* seq_lens,
                      int32_t n_pages, int32_t page_size, int32_t max_pages, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    return decode_cache("tt_attn_decode_q4", tt_cache_q4_page_bytes, attn_decode_q4_workspace, attn_decode_q4, desc, q, k_cache, v_cache, block_table, seq_lens, n_pages, page_size, max_pages, out, lse, workspace, workspace_bytes, stream);
}

size_t tt_cache_q8_page_bytes(int32_t page_size, int32_t D) {
    if ((D != 64 && D != 128) || page_size < 16 || page_size % 16) return 0;
    return (size_t)page_size * D + (size_t)(page_size / 16 + 31) / 32 * 32;
}

int tt_cache_append_q8(const void* k, const void* v, const int32_t* slots, int32_t T, int32_t Hkv, int32_t D, int32_t dtype, const int64_t* k_stride,
                       const int64_t* v_stride, void* k_cache, void* v_cache, int32_t n_pages, int32_t page_size, void* stream) {
    return append_to_cache("tt_cache_append_q8", tt_cache_q8_page_bytes(page_size, D), cache_append_q8, k, v, slots, T, Hkv, D, dtype, k_stride, v_stride, k_cache, v_cache, n_pages, page_size, stream);
}

int tt_cache_read_q8(const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* cu_lens, int32_t B, int32_t Hkv, int32_t D,
                     int32_t n_pages, int32_t page_size, int32_t max_pages, int32_t total, void* k, void* v, void* stream) {
    return read_from_cache("tt_cache_read_q8", tt_cache_q8_page_bytes(page_size, D), cache_read_q8, k_cache, v_cache, block_table, cu_lens, B, Hkv, D, n_pages, page_size, max_pages, total, k, v, stream);
}

size_t tt_attn_decode_q8_workspace_bytes(const tt_attn_desc* desc) {
    AttnArgs a;
    return resolve_cache("tt_attn_decode_q8_workspace_bytes", desc, &a) == TT_OK ? attn_decode_q8_workspace(a) : 0;
}
int tt_attn_decode_q8(const tt_attn_desc* desc, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* seq_lens,
                      int32_t n_pages, int32_t page_size, int32_t max_pages, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    return decode_cache("tt_attn_decode_q8", tt_cache_q8_page_bytes, attn_decode_q8_workspace, attn_decode_q8, desc, q, k_cache, v_cache, block_table, seq_lens, n_pages, page_size, max_pages, out, lse, workspace, workspace_bytes, stream);
}

int tt_rotary(const tt_rotary_desc* d, const void* q, const void* k, const int32_t* positions, const double* inv_freq, const int32_t* axes, int32_t backward,
              void* q_out, void* k_out, void* stream) {
    const char* who = "tt_rotary";
    int rc = rotary_desc_args(who, d, true, k != nullptr);
    if (rc != TT_OK) return rc;
    if ((k == nullptr) != (k_out == nullptr)) return fail(TT_ERR_NULL, "%s: k and k_out go together", who);
    if (d->B == 0 || d->S == 0) return TT_OK;
    if (!q || !q_out || !positions || !inv_freq) return fail(TT_ERR_NULL, "%s: null pointer", who);
    const Heads h(d, q, k, q_out, k_out, element(d));
    if ((rc = h.check(who, d)) != TT_OK || (rc = rotary_spans(who, h, d, positions, inv_freq, axes)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    RotaryArgs a = rotary_args(d, q, k, positions, inv_freq, axes, q_out, k_out);
    a.back = backward != 0;
    const cudaError_t e = rotary(a, d->dtype == TT_BF16, d->interleaved != 0, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_rotary: launch");
}

int tt_norm_rotary(const tt_rotary_desc* d, const void* q, const void* k, const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps,
                   const int32_t* positions, const double* inv_freq, const int32_t* axes, void* q_out, void* k_out, void* stream) {
    const char* who = "tt_norm_rotary";
    int rc = rotary_desc_args(who, d, true, k != nullptr);
    if (rc != TT_OK || (rc = norm_args(who, d, weight_dtype, eps)) != TT_OK) return rc;
    if ((k == nullptr) != (k_out == nullptr)) return fail(TT_ERR_NULL, "%s: k and k_out go together", who);
    if (d->B == 0 || d->S == 0) return TT_OK;
    if (!q || !q_out || !positions || !inv_freq || !q_weight || (k && !k_weight)) return fail(TT_ERR_NULL, "%s: null pointer", who);
    const Heads h(d, q, k, q_out, k_out, element(d));
    if ((rc = h.check(who, d)) != TT_OK || (rc = rotary_spans(who, h, d, positions, inv_freq, axes)) != TT_OK) return rc;
    if ((rc = weight_spans(who, h, d, q_weight, k_weight, weight_dtype)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    NormRotaryArgs a = {};
    a.r = rotary_args(d, q, k, positions, inv_freq, axes, q_out, k_out);
    a.w[0] = q_weight; a.w[1] = k_weight; a.w_bf16 = weight_dtype == TT_BF16; a.eps = eps;
    const cudaError_t e = norm_rotary(a, d->dtype == TT_BF16, d->interleaved != 0, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_norm_rotary: launch");
}

size_t tt_norm_rotary_bwd_workspace_bytes(const tt_rotary_desc* d) {
    return d && d->D > 0 && d->D <= 256 && check_device() == TT_OK ? norm_rotary_backward_workspace(d->D) : 0;
}

int tt_norm_rotary_bwd(const tt_rotary_desc* d, const void* dq, const void* dk, const void* q, const void* k, const int64_t* q_stride, const int64_t* k_stride,
                       const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps, const int32_t* positions, const double* inv_freq,
                       const int32_t* axes, void* dq_out, void* dk_out, void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "tt_norm_rotary_bwd";
    const bool two = dk_weight != nullptr;   // (no rows have no address)
    int rc = rotary_desc_args(who, d, true, two);
    if (rc != TT_OK || (rc = norm_args(who, d, weight_dtype, eps)) != TT_OK) return rc;
    const bool empty = d->B == 0 || d->S == 0;
    if (!dq_weight || (!empty && (!dq || !dq_out || !q || !positions || !inv_freq || !q_weight || !q_stride))) return fail(TT_ERR_NULL, "%s: null pointer", who);
    if (!empty && ((dk == nullptr) == two || (dk_out == nullptr) == two || (two && (!k || !k_weight || !k_stride))))
        return fail(TT_ERR_NULL, "%s: dk, k, k_weight, dk_out and dk_weight go together", who);
    const size_t size = element(d), w_size = weight_dtype == TT_BF16 ? 2 : 4, w = (size_t)d->D * w_size;
    if (((uintptr_t)dq_weight | (uintptr_t)dk_weight) % w_size) return fail(TT_ERR_BAD_SHAPE, "%s: weights must be multiples of their element size", who);
    const Span sums[3] = {{dq_weight, w, "dq_weight"}, {dk_weight, w, "dk_weight"}, {workspace, workspace_bytes, "workspace"}};
    for (int i = 1; i < 3; ++i)
        for (int j = 0; j < i; ++j)
            if (overlap(sums[i], sums[j])) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, sums[i].name, sums[j].name);
    NormRotaryArgs a = {};
    if (!empty) {
        const Heads h(d, dq, dk, dq_out, dk_out, size);
        if ((rc = h.check(who, d)) != TT_OK || (rc = rotary_spans(who, h, d, positions, inv_freq, axes)) != TT_OK) return rc;
        if ((rc = weight_spans(who, h, d, q_weight, k_weight, weight_dtype)) != TT_OK) return rc;
        for (int i = 0; i < 3; ++i)
            if (q_stride[i] < 0 || (two && k_stride[i] < 0)) return fail(TT_ERR_BAD_SHAPE, "%s: negative stride", who);
        if (((uintptr_t)q | (two ? (uintptr_t)k : 0)) % size) return fail(TT_ERR_BAD_SHAPE, "%s: pointers must be multiples of the element size", who);
        const int64_t* st[2] = {q_stride, k_stride};
        const void* x[2] = {q, k};
        for (int j = 0; j < h.count; ++j) {
            const Rows in(x[j], st[j], h.n[j], d->D, size, j ? "k" : "q");
            for (int i = 0; i < h.count; ++i)
                if (rows_meet(h.out[i], in, d->D, size)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, h.out[i].span.name, in.span.name);
            for (const Span& y : sums)
                if (overlap(y, in.span) || overlap(y, h.in[j].span) || overlap(y, h.out[j].span))
                    return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps the heads or their gradients", who, y.name);
            for (int i = 0; i < 3; ++i) a.in_stride[j][i] = st[j][i];
            a.in[j] = x[j];
        }
        const Span also[] = {{q_weight, w, "q_weight"}, {two ? k_weight : nullptr, w, "k_weight"}, {inv_freq, (size_t)d->R / 2 * 8, "inv_freq"},
                             {axes, (size_t)d->R / 2 * 4, "axes"}, positions_span(d, positions)};
        for (const Span& x_ : also)
            for (const Span& y : sums)
                if (overlap(x_, y)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, y.name, x_.name);
    }
    if ((rc = check_device()) != TT_OK) return rc;
    const size_t need = norm_rotary_backward_workspace(d->D);
    if (!workspace || workspace_bytes < need) return fail(TT_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, workspace_bytes);
    if ((uintptr_t)workspace & 255) return fail(TT_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    a.r = rotary_args(d, dq, dk, positions, inv_freq, axes, dq_out, dk_out);
    a.r.heads[0] = d->H; a.r.heads[1] = two ? d->Hkv : 0;
    a.r.back = 1;
    a.w[0] = q_weight; a.w[1] = k_weight; a.w_bf16 = weight_dtype == TT_BF16; a.eps = eps;
    a.dw[0] = dq_weight; a.dw[1] = dk_weight;
    const cudaError_t e = norm_rotary_backward(a, d->dtype == TT_BF16, d->interleaved != 0, workspace, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_norm_rotary_bwd: launch");
}

int tt_cache_append_rotary(const tt_rotary_desc* d, const void* q, const void* k, const void* v, const int64_t* v_stride, const int32_t* slots, const int32_t* positions,
                           const double* inv_freq, const int32_t* axes, const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps, void* q_out,
                           void* k_out, void* k_pool, void* v_pool, int32_t n_pages, int32_t page_size, void* stream) {
    const char* who = "tt_cache_append_rotary";
    int rc = rotary_desc_args(who, d, q != nullptr, true);
    if (rc != TT_OK) return rc;
    const bool normed = k_weight != nullptr;
    if (normed && (rc = norm_args(who, d, weight_dtype, eps)) != TT_OK) return rc;
    if (d->B != 1) return fail(TT_ERR_BAD_SHAPE, "%s: B=%d, packed tokens are one batch entry", who, d->B);
    if (d->D != 64 && d->D != 128) return fail(TT_ERR_UNSUPPORTED, "%s: head dim 64 or 128 only, got %d", who, d->D);
    if (page_size < 1 || n_pages < 0) return fail(TT_ERR_BAD_SHAPE, "%s: n_pages=%d page_size=%d", who, n_pages, page_size);
    if ((int64_t)n_pages * page_size >= (1LL << 31)) return fail(TT_ERR_BAD_SHAPE, "%s: pages of %d x %d tokens, at most 2^31 - 1", who, n_pages, page_size);
    if ((q == nullptr) != (q_out == nullptr)) return fail(TT_ERR_NULL, "%s: q and q_out go together", who);
    if (q && normed != (q_weight != nullptr)) return fail(TT_ERR_NULL, "%s: q_weight and k_weight go together", who);
    if (!q) q_weight = nullptr;
    if (normed && ((uintptr_t)q_weight | (uintptr_t)k_weight) % (weight_dtype == TT_BF16 ? 2 : 4))
        return fail(TT_ERR_BAD_SHAPE, "%s: weights must be multiples of their element size", who);
    if (!v_stride) return fail(TT_ERR_NULL, "%s: null strides", who);
    if (d->S == 0) return TT_OK;
    if (!k || !v || !slots || !positions || !inv_freq || (n_pages && (!k_pool || !v_pool))) return fail(TT_ERR_NULL, "%s: null pointer", who);
    const size_t size = element(d);
    const int64_t vs[3] = {0, v_stride[1], v_stride[0]};
    const int nk[3] = {1, d->Hkv, d->S}, nq[3] = {1, d->H, d->S};
    for (int i = 0; i < 3; ++i)
        if ((q && (d->q_stride[i] < 0 || d->q_out_stride[i] < 0)) || d->k_stride[i] < 0 || (k_out && d->k_out_stride[i] < 0) || vs[i] < 0 || (i < 2 && d->pos_stride[i] < 0))
            return fail(TT_ERR_BAD_SHAPE, "%s: negative stride", who);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % size || ((uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)k_pool | (uintptr_t)v_pool) % 2)
        return fail(TT_ERR_BAD_SHAPE, "%s: pointers must be multiples of the element size", who);
    if ((q && !rows_apart(d->q_out_stride, nq, d->D)) || (k_out && !rows_apart(d->k_out_stride, nk, d->D)))
        return fail(TT_ERR_BAD_SHAPE, "%s: rows of an output overlap", who);
    const Rows in[3] = {{q, d->q_stride, nq, d->D, size, "q"}, {k, d->k_stride, nk, d->D, size, "k"}, {v, vs, nk, d->D, size, "v"}};
    const Rows out[2] = {{q_out, d->q_out_stride, nq, d->D, 2, "q_out"}, {k_out, d->k_out_stride, nk, d->D, 2, "k_out"}};
    const size_t pool = (size_t)n_pages * d->Hkv * page_size * d->D * 2, w = (size_t)d->D * (weight_dtype == TT_BF16 ? 2 : 4);
    const Span pools[2] = {{k_pool, pool, "k_pool"}, {v_pool, pool, "v_pool"}};
    const Span also[] = {positions_span(d, positions), {inv_freq, (size_t)d->R / 2 * 8, "inv_freq"}, {axes, (size_t)d->R / 2 * 4, "axes"},
                         {slots, (size_t)d->S * 4, "slots"}, {q_weight, w, "q_weight"}, {k_weight, w, "k_weight"}};
    // Queries and keys may be turned in place, where the types are the same; else outputs lie apart from everything.
    for (int i = 0; i < 2; ++i) {
        if (!out[i].span.p) continue;
        for (int j = 0; j < 3; ++j) {
            if (!in[j].span.p || (i == j && size == 2 && in_place(out[i], in[j]))) continue;
            if (size == 2 ? rows_meet(out[i], in[j], d->D, size) : overlap(out[i].span, in[j].span))
                return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].span.name, in[j].span.name);
        }
        for (const Span& x : also)
            if (overlap(out[i].span, x)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].span.name, x.name);
        for (const Span& x : pools)
            if (overlap(out[i].span, x)) return fail(TT_ERR_BAD_SHAPE, "%s: %s overlaps %s", who, out[i].span.name, x.name);
    }
    if (q && k_out && rows_meet(out[0], out[1], d->D, 2)) return fail(TT_ERR_BAD_SHAPE, "%s: q_out overlaps k_out", who);
    const Span ins[] = {in[0].span, in[1].span, in[2].span};
    if ((rc = check_overlap(who, pools, 2, ins, 3)) != TT_OK || (rc = check_overlap(who, pools, 2, also, 6)) != TT_OK || (rc = check_device()) != TT_OK) return rc;
    NormRotaryArgs a = {};
    a.r = rotary_args(d, q, k, positions, inv_freq, axes, q_out, k_out);
    a.w[0] = q_weight; a.w[1] = k_weight; a.w_bf16 = weight_dtype == TT_BF16; a.eps = eps;
    a.v = v; a.v_stride[0] = v_stride[0]; a.v_stride[1] = v_stride[1];
    a.slots = slots;
    a.pool[0] = k_pool; a.pool[1] = v_pool; a.n_slots = n_pages * page_size; a.page = page_size;
    const cudaError_t e = cache_append_rotary(a, d->dtype == TT_BF16, d->interleaved != 0, (cudaStream_t)stream);
    return e == cudaSuccess ? TT_OK : cuda_fail(e, "tt_cache_append_rotary: launch");
}

}  // extern "C"
