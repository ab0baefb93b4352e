/*
 * tt_attn.h -- C ABI of the B200 (sm_100a) attention kernels for TinyTensor.
 *
 * This is the boundary a host framework binds: plain pointers and sizes, no C++ or
 * torch types.  The reference project (TinyTensor) reaches its GPU code through C++
 * free functions over `TinyTensor<T>` bound with pybind11; each entry point below names
 * the reference interface it sits under.  Paths are relative to the reference project
 * root (`Task3/Tinytensor/`).
 *
 * Conventions
 *   - All tensors are dense row-major, contiguous: q/out/dout/dq `[B,H,S,D]`,
 *     k/v/dk/dv `[B,H,L,D]`, lse `[B,H,S]` (float, natural log of the softmax
 *     denominator including the row maximum).
 *   - Pointers are DEVICE pointers unless the function name ends in `_host`.
 *   - `stream` is a `cudaStream_t` passed as `void*`; calls are asynchronous on it.
 *   - `scale <= 0` selects `1/sqrt(D)`.
 *   - causal: query i attends to keys j <= i + (L - S) (bottom-right aligned);
 *     causal with L < S is rejected (some rows would have no key).
 *   - Every function returns a `tt_status`; none throws or aborts.  A human-readable
 *     message for the last failure on the calling thread is at `tt_last_error()`.
 *   - There is no CPU path: a call on a machine without a usable sm_100 device returns
 *     TT_ERR_BAD_DEVICE.
 */
#ifndef TT_ATTN_H
#define TT_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

typedef enum tt_status {
    TT_OK = 0,
    TT_ERR_NULL = 1,        /* a required pointer is null */
    TT_ERR_BAD_SHAPE = 2,   /* non-positive extent, unsupported head dim, causal with L < S */
    TT_ERR_BAD_DTYPE = 3,
    TT_ERR_BAD_DEVICE = 4,  /* no CUDA device, or not compute capability 10.x */
    TT_ERR_WORKSPACE = 5,   /* workspace missing or smaller than *_workspace_bytes() */
    TT_ERR_CUDA = 6,        /* a CUDA runtime/driver call failed */
    TT_ERR_TIMEOUT = 7,     /* a bounded device-side wait expired (reported after a sync) */
    TT_ERR_UNSUPPORTED = 8,
    TT_ERR_NCCL = 9         /* the NCCL library is missing, or one of its calls failed */
} tt_status;

typedef enum tt_dtype { TT_F32 = 0, TT_BF16 = 1 } tt_dtype;

/* Problem description shared by every entry point. */
typedef struct tt_attn_desc {
    int32_t B, H;     /* batch, heads: B*H independent slices */
    int32_t S;        /* queries per slice */
    int32_t L;        /* keys/values per slice */
    int32_t D;        /* head dim: 1..256 (tensor-core path: 64 or 128, bf16) */
    int32_t dtype;    /* tt_dtype of q,k,v,out and gradients */
    int32_t causal;   /* 0 / 1 */
    float scale;      /* <= 0 -> 1/sqrt(D) */
    int32_t Hkv;      /* key/value heads; 0 or H: one per query head.  Hkv < H (H % Hkv == 0) is grouped
                       * (GQA / MQA) attention: k, v, dk, dv are [B,Hkv,L,D] and query head h reads
                       * key/value head h / (H/Hkv); dk, dv are summed over the group.  No counterpart
                       * in the reference. */
} tt_attn_desc;

/* ---- forward -------------------------------------------------------------------------
 * out = softmax(scale * q k^T [+ causal mask]) v, lse = log sum exp of the scaled scores.
 * Replaces the composition MatMul/Transpose/MulScalar/EWiseAdd/Exp/Summation/Reshape/
 * BroadcastTo/EWiseDiv/MatMul of optimizer/operators.py:194-199,234-242,289-298,323-340,
 * 348-380,388-408,416-429,464-470, and on the native side the cudaGemm + SoftmaxForward
 * sequence of src/Layers_kernels.cu:10-30 and src/Layers.cu:324-349.
 * `lse` may be null when no backward will follow.  Needs no workspace. */
int tt_attn_fwd(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                void* out, float* lse, void* stream);

/* ---- backward ------------------------------------------------------------------------
 * dq, dk, dv of sum(out * dout); `out` and `lse` are the forward's results.
 * Replaces the reverse sweep of optimizer/autodiff.py:33-61 over the gradient methods of
 * the ops listed above (operators.py:198-199,241-242,296-298,338-340,356-358,373-380,
 * 400-408,421-429,469-470).
 * Workspace: tt_attn_bwd_workspace_bytes() bytes of device memory, 256-byte aligned;
 * contents on entry are ignored. */
size_t tt_attn_bwd_workspace_bytes(const tt_attn_desc* desc);
int tt_attn_bwd(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                const void* out, const float* lse, const void* dout,
                void* dq, void* dk, void* dv,
                void* workspace, size_t workspace_bytes, void* stream);

/* The tensor-core backward (bf16, D = 64 or 128) exists twice.  Two passes (dk/dv with the keys resident,
 * then dq with the queries resident and the scores recomputed): seven GEMMs per tile pair, no atomics,
 * every result bit-reproducible.  One pass that produces dk, dv and dq together (five GEMMs), dq through
 * fp32 additions into the workspace; those arrive in no fixed order, so dq repeats to fp32 rounding (a few
 * 1e-7 relative) rather than bit for bit.  on = 1: always the two passes.  on = 0: whichever measured faster
 * for the shape, the single pass for problems of several key tiles per SM that each meet several query tiles and,
 * at D = 64, for few queries against many keys.  A process that never calls this gets the two passes for packed
 * batches and at D = 128, and at D = 64 what on = 0 gives.  Process-wide; no counterpart in
 * the reference, whose NumPy reverse sweep (optimizer/autodiff.py:33-61) is deterministic and
 * single-threaded. */
int tt_attn_bwd_set_deterministic(int on);

/* ---- single-query decode (S == 1) ----------------------------------------------------
 * The memory-bound case: every K and V row is streamed once.  Same mathematics as
 * tt_attn_fwd with S == 1, no mask.  bf16 at D = 128 or 64 with up to 16 query heads per key/value
 * head runs a tensor-core kernel whose accumulator rows are the keys (K and V tiles by TMA,
 * the group's query heads as 16 B-operand rows, one CTA per (key/value slice, key range));
 * other shapes a split-KV kernel with 16-byte loads.  With more than one key range per slice
 * a second small kernel merges the partial results.
 * Workspace: tt_attn_decode_workspace_bytes() bytes (partials), 256-byte aligned.
 * `lse` may be null. */
size_t tt_attn_decode_workspace_bytes(const tt_attn_desc* desc);
int tt_attn_decode(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                   void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream);

/* Decode for callers that cannot allocate device memory.  No counterpart in the reference:
 * it exists for hosts that run with a frozen memory map -- a real-time serving loop that
 * pre-allocated everything at start-up and may not touch the allocator again, or a plugin sandbox
 * whose policy forbids cudaMalloc -- and therefore cannot supply the partials workspace
 * tt_attn_decode wants.  It always runs the split-KV kernels named above (tt_attn_decode prefers the
 * tensor-core decode kernel), so its results match tt_attn_decode within the bf16
 * tolerance, bit for bit where both take the same
 * kernels; the split-KV partials go to an 8 MiB array built into the library's device image (each
 * GPU that loads the library keeps those 8 MiB until the process exits).  The call itself performs
 * no cudaMalloc/cudaFree and calls no allocating library routine; q, k, v, out (and lse) are still the caller's.
 *   - bf16, D = 64 or 128, S = 1 only; problems whose partials exceed the array are refused
 *     with TT_ERR_WORKSPACE and a message naming both sizes (B*H*(D+2)*4*splits bytes; e.g.
 *     B*H up to ~4000 slices at D = 128 with 4 key ranges each).
 *   - The first call on each device looks up the array's device address (one runtime query);
 *     make that first call outside any stream capture.
 *   - All calls on a device share the one array, and it keeps whatever the previous call
 *     left; nothing in it needs clearing because each call overwrites every partial it
 *     later reads.  Two calls that overlap on the GPU (different streams) race on it:
 *     serialise them. */
int tt_attn_decode_static(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                          void* out, float* lse, void* stream);

/* ---- padded batches -------------------------------------------------------------------------
 * tt_attn_fwd / tt_attn_bwd with a key padding length per batch entry (no counterpart in the
 * reference): kv_lens is a device array of B int32; batch entry b attends to its first kv_lens[b]
 * keys (clamped to 1..L), the rest of its k, v rows is padding.  dk, dv rows of padded keys are
 * zero.  Query rows are all computed (give padded queries a zero dout).  The causal mask keeps its
 * alignment to the full L.  Padding rows must hold finite values (zeros are customary): a masked
 * probability of exactly 0 still meets them in the P.V and dS.K products.  kv_lens == NULL is the
 * unpadded call. */
int tt_attn_fwd_padded(const tt_attn_desc* desc, const void* q, const void* k, const void* v, const int32_t* kv_lens,
                       void* out, float* lse, void* stream);
int tt_attn_bwd_padded(const tt_attn_desc* desc, const void* q, const void* k, const void* v, const int32_t* kv_lens,
                       const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                       void* workspace, size_t workspace_bytes, void* stream);

/* ---- packed variable-length batches ----------------------------------------------------------
 * n_seq sequences of different lengths stored back to back, token-major, without padding (no counterpart
 * in the reference, whose tensors are dense [B,H,S,D], src/TinyTensor.h:14-17): q, out, dout, dq are
 * [total_q, H, D]; k, v, dk, dv [total_k, Hkv, D]; lse [H, total_q].  cu_q, cu_k: device arrays of
 * n_seq + 1 int32, cumulative token counts (cu[0] = 0, cu[n_seq] = total): sequence b owns query tokens
 * [cu_q[b], cu_q[b+1]) and key tokens [cu_k[b], cu_k[b+1]).  max_q, max_k: upper bounds of the longest
 * sequence (host values: the two-pass backward numbers its work for them, the forward orders its work by them; the
 * kernels read the real lengths from cu_q / cu_k).
 * Every sequence is its own attention problem with the conventions above (causal: bottom-right aligned
 * per sequence; a row that sees no key -- an empty key sequence, or causal with fewer keys than queries --
 * gets out = 0, lse = -inf and zero gradients).  bf16 with D = 64 or 128 only (tensor-core kernels);
 * anything else returns TT_ERR_UNSUPPORTED.  The backward runs the two-pass kernels (bit-reproducible) unless
 * tt_attn_bwd_set_deterministic(0) has allowed the single pass.
 * Workspace: tt_attn_bwd_varlen_workspace_bytes(), 256-byte aligned: 8 bytes per query row and head for the two
 * passes.  Where the single pass is allowed and would be taken, H * (total_q / 128 + n_seq) * 128 * (D + 2) * 4
 * bytes, at most 2 * total_q * H * (D + 2) * 4; a call that is given less than that, but enough for the two
 * passes, takes them. */
typedef struct tt_varlen_desc {
    int32_t n_seq, H, Hkv;   /* Hkv: 0 or H, or a divisor of H (grouped heads) */
    int32_t D, dtype, causal;
    float scale;             /* <= 0 -> 1/sqrt(D) */
    int32_t max_q, max_k;
    int64_t total_q, total_k;
} tt_varlen_desc;
int tt_attn_fwd_varlen(const tt_varlen_desc* desc, const void* q, const void* k, const void* v, const int32_t* cu_q,
                       const int32_t* cu_k, void* out, float* lse, void* stream);
size_t tt_attn_bwd_varlen_workspace_bytes(const tt_varlen_desc* desc);
int tt_attn_bwd_varlen(const tt_varlen_desc* desc, const void* q, const void* k, const void* v, const int32_t* cu_q,
                       const int32_t* cu_k, const void* out, const float* lse, const void* dout, void* dq, void* dk,
                       void* dv, void* workspace, size_t workspace_bytes, void* stream);

/* ---- decode over a paged and/or ragged key/value cache -----------------------------------
 * tt_attn_decode for serving-style caches (no counterpart in the reference).  bf16, D = 64 or
 * 128, S = 1; desc->L is the longest sequence any batch entry may have.
 *   block_table != NULL: k_pool, v_pool are page pools [pages, Hkv, page_size, D]; key r of batch
 *       entry b is row r % page_size of page block_table[b * max_pages + r / page_size]
 *       (device array of B * max_pages int32); page_size * max_pages >= L.
 *   block_table == NULL: k_pool, v_pool are dense [B, Hkv, L, D] as in tt_attn_decode.
 *   seq_lens != NULL: device array of B int32, batch entry b attends to its first seq_lens[b]
 *       keys (clamped to 0..L); an entry with no keys gets out = 0 and lse = -inf.
 * Grouped heads (desc->Hkv < H) read each key/value row once for the whole group: groups of up to
 * 16 on the tensor-core decode kernel, as in tt_attn_decode, larger ones on the tensor-core forward
 * kernel.  Over a paged cache the tensor-core
 * kernels need a page_size that divides 128 or is a multiple of it (>= 8) and gather the pages by
 * TMA; other page sizes take the split-KV kernel.  Rows that no sequence owns never reach the
 * result and may hold anything.  Workspace: tt_attn_decode_workspace_bytes(desc). */
int tt_attn_decode_paged(const tt_attn_desc* desc, const void* q, const void* k_pool, const void* v_pool,
                         const int32_t* block_table, const int32_t* seq_lens, int32_t page_size, int32_t max_pages,
                         void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream);

/* ---- page tables of a paged cache ---------------------------------------------------------
 * The block table and the slots of new tokens, made on the GPU from the requests' lengths (no counterpart in the reference).
 * block_table is [B, max_pages]; request b's first seq_lens[b] tokens lie in its columns 0 .. ceil(seq_lens[b] / page_size) - 1.
 * free_pages holds *n_free page numbers (an array of free_capacity), used from its end.  All arrays are device int32.
 *
 * tt_cache_extend: new_lens[b] more tokens for request b.  Requests are served in their order until the next one's tokens
 * exceed max_tokens in all or its pages exceed *n_free; that one and those behind it get nothing.  A request with a negative
 * count, or one whose tokens do not fit its max_pages, gets nothing and keeps none from being served.
 *   block_table   the new pages' columns are written, nothing else
 *   seq_lens_out  [B] lengths with the new tokens (seq_lens where a request got nothing)
 *   n_free_out    [1] what is left of *n_free
 *   cu_new        [B + 1] cumulative counts of the tokens served: request b's are rows [cu_new[b], cu_new[b + 1])
 *   slots         [max_tokens] page * page_size + row in the page, by packed row; -1 behind the last row
 *                 (and where block_table holds a negative page for a token of a page that was there before)
 *   positions     [max_tokens] each row's place in its sequence; 0 behind the last row
 * free_pages is not written: the pages taken are those at *n_free_out and above.
 *
 * tt_cache_release: the pages of the requests with done[b] != 0 (bytes) go back: free_pages[*n_free ..] gets them in order of
 * request and column (none beyond free_capacity), seq_lens_out is 0 there, n_free_out counts them.  block_table is only read.
 * Negative entries are no pages and are left out; as many places of free_pages behind n_free_out may then have been written.
 *
 * Outputs must not overlap inputs or each other, except block_table and free_pages as said.  B is at most 16384, and slots
 * fit 32 bits (pages * page_size < 2^31).  Negative lengths of done requests count as 0, ones beyond a row as the whole row. */
int tt_cache_extend(int32_t* block_table, const int32_t* seq_lens, const int32_t* new_lens, const int32_t* free_pages,
                    const int32_t* n_free, int32_t B, int32_t page_size, int32_t max_pages, int32_t free_capacity,
                    int32_t max_tokens, int32_t* seq_lens_out, int32_t* n_free_out, int32_t* cu_new, int32_t* slots,
                    int32_t* positions, void* stream);
int tt_cache_release(const int32_t* block_table, const int32_t* seq_lens, const uint8_t* done, int32_t* free_pages,
                     const int32_t* n_free, int32_t B, int32_t page_size, int32_t max_pages, int32_t free_capacity,
                     int32_t* seq_lens_out, int32_t* n_free_out, void* stream);

/* ---- key/value cache in 4 bits --------------------------------------------------------------
 * k_cache, v_cache: [n_pages, Hkv, tt_cache_q4_page_bytes(page_size, D)] bytes each, 16-byte aligned; D 64 or 128, page_size a
 * multiple of 16.  A page holds, for one key/value head, [page_size][D / 2] bytes (channel 2j in the low half of byte j) and then
 * [page_size][D / 32] scale codes, one for 32 channels: 4.25 bits a value.  Code c stands for the scale s = half(c << 7) / 8, i.e. five bits
 * of exponent and three of mantissa; a value is (n - 8) s with n in 0 .. 15, which bf16 holds exactly.  A cache is below 2^37 bytes,
 * and has less than 2^31 tokens.
 *
 * tt_cache_append_q4: T new tokens' keys and values [T, Hkv, D] (float or bf16, channels next to each other, element strides
 * {token, head}) into their slots (page * page_size + row, as from tt_cache_extend).  A slot that is negative or behind the last page is
 * passed over; no two tokens may have one slot (what such a slot then holds is of either, and may be of both).  k and v must not lie
 * in the cache.  Per group: s is
 * the smallest scale with 7.5 s >= max |x|, n = rint(x / s) (ties to even) held to -8 .. 7, plus 8, so an error is at most s / 2.
 * The largest scale is 896: values beyond 6720 and infinities become the largest.  A group with a NaN reads as NaN.
 *
 * tt_cache_read_q4: the first cu_lens[b + 1] - cu_lens[b] tokens of each sequence as packed bf16 k, v [total, Hkv, D] (what
 * tt_attn_fwd_varlen takes); sequence b's are rows [cu_lens[b], cu_lens[b + 1]), found by block_table [B, max_pages].  cu_lens
 * counts up from 0.  Rows from cu_lens[B] on are left as they were; rows whose page is not one of the n_pages, or lies behind the
 * table's width, are 0.  k and v must not overlap each other or an input. */
size_t tt_cache_q4_page_bytes(int32_t page_size, int32_t D);   /* 0: not supported */
int tt_cache_append_q4(const void* k, const void* v, const int32_t* slots, int32_t T, int32_t Hkv, int32_t D, int32_t dtype,
                       const int64_t* k_stride, const int64_t* v_stride, void* k_cache, void* v_cache, int32_t n_pages,
                       int32_t page_size, void* stream);
int tt_cache_read_q4(const void* k_cache, const void* v_cache, const int32_t* block_table, const int32_t* cu_lens, int32_t B,
                     int32_t Hkv, int32_t D, int32_t n_pages, int32_t page_size, int32_t max_pages, int32_t total, void* k, void* v,
                     void* stream);

/* Decode over a 4-bit cache: tt_attn_decode_paged with q and out bf16 [B, H, 1, D] and the cache as above.
 *   block_table    [B, max_pages]; key r of batch entry b is row r % page_size of page block_table[b, r / page_size].  Keys of a
 *                  page that is not one of the n_pages, or of a column behind max_pages, count as absent.
 *                  NULL: batch entry b has page b to itself (page_size >= desc->L, n_pages >= B).
 *   seq_lens       [B] or NULL (desc->L each), clamped to 0 .. desc->L; an entry without keys gets out = 0, lse = -inf
 * desc: dtype TT_BF16, S = 1, D 64 or 128, L the longest sequence there may be, at most 2^30; any group H / Hkv.  `lse` may be NULL.
 * q may be of any finite size, as long as scale * q is finite in 32 bits and scores stay below 2^127.
 * out, lse and the workspace must not overlap each other or an input, so `out` cannot be `q`.  A group of more than 16 query heads
 * reads the cache once for each 16 of them.
 * Products are exact in what the cache holds; probabilities are rounded to 11 bits, sums are 32-bit.  Results repeat to the bit.
 * Workspace: tt_attn_decode_q4_workspace_bytes(desc) bytes, 256-byte aligned, contents ignored; 0 (and NULL) where L is at most 128. */
size_t tt_attn_decode_q4_workspace_bytes(const tt_attn_desc* desc);
int tt_attn_decode_q4(const tt_attn_desc* desc, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                      const int32_t* seq_lens, int32_t n_pages, int32_t page_size, int32_t max_pages, void* out, float* lse,
                      void* workspace, size_t workspace_bytes, void* stream);

/* ---- rotary positions ------------------------------------------------------------------------
 * Query and key heads turned by their tokens' positions (no counterpart in the reference).  Of a head's D channels the first
 * R form R / 2 pairs; pair i of a token at position p on axis a = axes[i] turns by p * inv_freq[i]:
 *     (x1, x2) -> scale * (x1 cos - x2 sin, x2 cos + x1 sin)
 * Pairs are halves (channels i and i + R / 2) or, with `interleaved`, neighbours (2i and 2i + 1); channels from R on are copied.
 * `backward` turns the other way (sin -> -sin): the gradient of the call with the same arguments, which is linear in x.
 * Angles are taken in 64 bits and reduced to one turn before their sine and cosine, products are 32-bit, outputs rounded once.
 *   q, k           [B, heads, S, D] at element strides {batch, head, row} of their own, channels next to each other; inputs may
 *                  repeat (stride 0), outputs may not.  An output may be its input (same pointer and strides), else the two must not
 *                  overlap, and no output what positions, inv_freq and axes span.  k and k_out are both null where there is one
 *                  tensor only.  Packed tokens [T, H, D]: B = 1, S = T.
 *   positions      int32, [n_axes, B, S] at strides pos_stride {axis, batch}, rows next to each other; any int32 value
 *   inv_freq       [R / 2] double, angle per position;  axes: [R / 2] int32 in 0 .. n_axes - 1 (others are taken as the nearest),
 *                  or null: all of axis 0
 * D at most 256, R even, dtype TT_F32 or TT_BF16.  Accesses are of up to 16 bytes, as pointers, strides and R allow. */
typedef struct tt_rotary_desc {
    int32_t B, S, H, Hkv, D, R, n_axes, dtype, interleaved;
    float scale;
    int64_t q_stride[3], k_stride[3], q_out_stride[3], k_out_stride[3];
    int64_t pos_stride[2];
} tt_rotary_desc;
int tt_rotary(const tt_rotary_desc* desc, const void* q, const void* k, const int32_t* positions, const double* inv_freq,
              const int32_t* axes, int32_t backward, void* q_out, void* k_out, void* stream);

/* ---- row softmax ------------------------------------------------------------------------
 * out[r,:] = softmax(in[r,:]) over `cols`, row maximum subtracted; rows = product of the leading
 * axes.  One launch that reads and writes every element once; replaces SoftmaxForward of
 * src/Layers.cu:324-349 with its five launches and per-row Thrust loops
 * (src/Layers_kernels.cu:189-257).  The backward, dx = y * (dy - sum(dy*y)), has no native
 * counterpart in the reference (its NumPy form is the Softmax part of optimizer/operators.py:
 * 610-626).  dtype: TT_F32 or TT_BF16 (fp32 arithmetic either way). */
int tt_softmax_fwd(const void* in, void* out, int64_t rows, int32_t cols, int32_t dtype, void* stream);
int tt_softmax_bwd(const void* y, const void* dy, void* dx, int64_t rows, int32_t cols, int32_t dtype, void* stream);

/* ---- fully connected layer ------------------------------------------------------------------
 * y[rows,out] = x[rows,in] . w[in,out] + bias[out]  (bias may be NULL), all row-major; replaces
 * FcForward of src/Layers.cu:9-40 (cublasSgemm through a handle created and destroyed per call
 * plus a rank-1 GEMM for the bias, src/Layers_kernels.cu:10-30).  tt_fc_bwd replaces FcBackward
 * of src/Layers.cu:42-79: dx = dy . w^T, dw = x^T . dy, db = column sums of dy (db_scalar != 0:
 * one value, the sum over all of dy, for the reference's single-value bias); each of dx, dw, db
 * may be NULL and is then skipped.  bf16 with in % 8 == 0 and out % 8 == 0 runs the tcgen05
 * kernel (fp32 accumulation), float of any shape a tcgen05 kernel on three bf16 parts per value,
 * other shapes an fp32 SIMT kernel; tt_fc_path says which (1 = tensor cores).  The workspace is only
 * needed for db. */
int tt_fc_fwd(const void* x, const void* w, const void* bias, void* y, int64_t rows, int32_t in_features,
              int32_t out_features, int32_t dtype, void* stream);
size_t tt_fc_bwd_workspace_bytes(int64_t rows, int32_t in_features, int32_t out_features, int32_t dtype);
int tt_fc_bwd(const void* x, const void* w, const void* dy, void* dx, void* dw, void* db, int32_t db_scalar, int64_t rows,
              int32_t in_features, int32_t out_features, int32_t dtype, void* workspace, size_t workspace_bytes,
              void* stream);
int tt_fc_path(int64_t rows, int32_t in_features, int32_t out_features, int32_t dtype);

/* ---- host-buffer calls (what the reference's Python ops do around each native op:
 * upload NumPy -> run -> download, optimizer/operators.py:502-512) ----------------------
 * Pointers are HOST pointers (pinned memory gives the best copy rate).  Device buffers
 * come from the pool below; the call uploads, runs, downloads and synchronises. */
int tt_attn_fwd_host(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                     void* out, float* lse);
int tt_attn_bwd_host(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                     const void* out, const float* lse, const void* dout,
                     void* dq, void* dk, void* dv);
int tt_attn_decode_host(const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                        void* out, float* lse);
/* One training step from host buffers: forward and backward of every slice, with the slices cut
 * into chunks that flow through an upload stream, a compute stream and a download stream, so
 * the PCIe transfers of both directions overlap the kernels (use pinned host memory; with
 * pageable memory the copies serialise).  What the Python autograd op does in two calls
 * (compute, then gradient with the tensors kept on the device, optimizer/operators.py:498-527
 * pattern of the reference) in one.  `lse` may be null. */
int tt_attn_fwd_bwd_host(const tt_attn_desc* desc, const void* q, const void* k, const void* v, const void* dout,
                         void* out, float* lse, void* dq, void* dk, void* dv);

/* ---- pooled device storage -----------------------------------------------------------
 * Replaces the per-object cudaMalloc/cudaFree of src/Tinytensor.cu:17-22,85-93: freed
 * blocks go to size-bucketed free lists of the current device and are reused. */
int tt_alloc(size_t bytes, void** out_ptr);
int tt_free(void* ptr);   /* does not synchronise: free a block only after the work that uses it has completed */
/* Host storage of the tensor class goes through the library too (plain malloc/free underneath), so that
 * the two rules below cover host and device buffers alike. */
int tt_host_alloc(size_t bytes, void** out_ptr);
int tt_host_free(void* ptr);
/* Shared ownership for zero-copy views (DLPack exports of the tensor class, src/bind_Tensor.cpp of the
 * reference has no such export): while a buffer is retained, tt_free / tt_host_free of it only mark it;
 * the block goes back to the pool (or the heap) when the last holder releases it.  So a tensor may be
 * resized, moved between host and device or destroyed while a view of its old buffer is alive. */
int tt_buffer_retain(void* ptr);
int tt_buffer_release(void* ptr);
int tt_pool_trim(void);                                     /* return cached blocks to the driver */
int tt_pool_stats(size_t* bytes_in_use, size_t* bytes_cached, uint64_t* n_driver_allocs);

/* ---- sharding of the B*H independent slices over ranks -------------------------------
 * Contiguous ranges, remainder spread over the first ranks; pure host arithmetic.
 * (The reference has no multi-GPU path; Task2/mnist.py:53-54 is torch DataParallel.) */
int tt_shard_range(int64_t n_slices, int32_t world, int32_t rank, int64_t* begin, int64_t* count);

/* ---- several GPUs: one process (or thread) per GPU, slices sharded, outputs all-gathered -------
 * The B*H slices are independent in forward and backward, so rank r of `world` owns the contiguous
 * range tt_shard_range(B*H, world, r) of them, keeps q, k, v, out, lse and the gradients of that
 * range in its own memory, and runs the single-GPU kernels on it; nothing crosses between GPUs on the
 * data path.  The one exchange is the all-gather that gives every rank the full `out` (and, if asked
 * for, full gradients): because [B,H,S,D] is contiguous in the slice index, each rank's shard is one
 * contiguous block of the full tensor and a single ncclAllGather lands it in place, no repacking.
 * The communicator owns one ncclComm_t and one side stream on its device: gathers run on the side
 * stream, ordered behind the kernels that produce their data, so the gather of `out` overlaps the
 * backward.  NCCL is bound at run time (dlopen of libnccl.so.2, or the library TT_NCCL_LIB names);
 * no kernel of this library reads another GPU's memory.
 * No counterpart in the reference, whose only multi-GPU construct is torch's nn.DataParallel around
 * a PyTorch model (Task2/mnist.py:53-54).
 *
 *   tt_mgpu_unique_id   rank 0 calls it and hands the TT_MGPU_ID_BYTES bytes to every rank by its own
 *                       means (a file, a socket, MPI, torch.distributed).
 *   tt_mgpu_init        collective over the ranks; binds the communicator to the CURRENT device.
 *   tt_mgpu_attn_fwd    desc describes the WHOLE problem (all B*H slices); the tensor arguments are this
 *                       rank's shard ([count,S,D] / [count/group,L,D] / [count,S]).  out_full, if not
 *                       null, is [B*H,S,D] on this device and receives every rank's out.
 *                       B*H must divide evenly by world, and a shard must hold whole groups of query
 *                       heads, else TT_ERR_UNSUPPORTED.  Kernels run on `stream`; returns at once.
 *   tt_mgpu_attn_bwd    same for the backward; dq_full / dk_full / dv_full (each may be null) receive
 *                       the all-gathered gradients, otherwise gradients stay with their owners.
 *                       Workspace: tt_mgpu_bwd_workspace_bytes(comm, desc), 256-byte aligned.
 *   tt_mgpu_wait        makes `stream` wait (on the device) for every gather issued so far.
 *   tt_mgpu_destroy     collective; frees the communicator, the side stream and the events. */
#define TT_MGPU_ID_BYTES 128
typedef struct tt_mgpu* tt_mgpu_t;
int tt_mgpu_unique_id(void* id_bytes);
int tt_mgpu_init(tt_mgpu_t* comm, int32_t world, int32_t rank, const void* id_bytes);
int tt_mgpu_destroy(tt_mgpu_t comm);
int tt_mgpu_shard(tt_mgpu_t comm, const tt_attn_desc* desc, int64_t* first_slice, int64_t* n_slices);
int tt_mgpu_attn_fwd(tt_mgpu_t comm, const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                     void* out, float* lse, void* out_full, void* stream);
size_t tt_mgpu_bwd_workspace_bytes(tt_mgpu_t comm, const tt_attn_desc* desc);
int tt_mgpu_attn_bwd(tt_mgpu_t comm, const tt_attn_desc* desc, const void* q, const void* k, const void* v,
                     const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                     void* dq_full, void* dk_full, void* dv_full, void* workspace, size_t workspace_bytes, void* stream);
int tt_mgpu_wait(tt_mgpu_t comm, void* stream);

/* ---- diagnostics ---------------------------------------------------------------------*/
const char* tt_last_error(void);
/* Number of kernels this library has launched in this process (for launch accounting). */
uint64_t tt_kernel_launch_count(void);
/* Name of the kernel family the given problem dispatches to: "tcgen05" or "simt". */
const char* tt_attn_fwd_path(const tt_attn_desc* desc);
const char* tt_attn_bwd_path(const tt_attn_desc* desc);
/* Reads (and clears) the device-side status word after synchronising `stream`:
 * TT_OK, or TT_ERR_TIMEOUT with details in tt_last_error(). */
int tt_check_device_status(void* stream);

/* Optional per-kernel timing: while enabled, every kernel launch of this library is
 * bracketed by CUDA events on its launching stream.  tt_profile_read() waits for the
 * recorded events and returns the accumulated device time and launch count of one kernel
 * family (ids 0 .. tt_profile_kernel_count()-1, names from tt_profile_kernel_name()). */
int tt_profile_enable(int on);
int tt_profile_reset(void);
int tt_profile_kernel_count(void);
const char* tt_profile_kernel_name(int kernel_id);
int tt_profile_read(int kernel_id, double* total_ms, uint64_t* launches);

/* Launches a one-warp kernel whose only wait can never be satisfied and whose wait budget is
 * `budget_cycles` SM cycles (at most 4e9).  The wait expires, the kernel returns normally, and the
 * next tt_check_device_status() reports TT_ERR_TIMEOUT (barrier id 99, iteration 7) and clears
 * the status word: a way to test the failure-reporting path without faulting or hanging a GPU. */
int tt_debug_wait_timeout(int64_t budget_cycles, void* stream);

/* Building-block self test of the tensor-core plumbing (TMA load -> tcgen05.mma from
 * shared memory -> tcgen05.ld, tcgen05.st -> tcgen05.mma with A in tensor memory and an
 * MN-major B).  a,b: bf16 [128,128] row-major; vt: bf16 [128,D] row-major (D = 64|128).
 * Outputs: s = a b^T as float [128,128]; o = bf16(s) vt as float [128,D]. */
int tt_debug_umma_probe(const void* a, const void* b, const void* vt, int32_t D,
                        float* s_out, float* o_out, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif
#endif /* TT_ATTN_H */
