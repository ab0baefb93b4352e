"""Attention calls over torch CUDA tensors.

torch is used for device memory and streams only: every call hands raw device pointers
to the C ABI, through the extension `_ttorch` (csrc/host/bind_torch.cpp), which checks the
arguments and allocates the outputs.  Where it finds that an argument does not fit it returns
None, and the `_explain_*` functions here say what is wrong.  Shapes follow the reference's row-major layout:
q/out `[B,H,S,D]`, k/v `[B,Hkv,L,D]` (Hkv = H, or a divisor of H for grouped heads), lse `[B,H,S]` fp32.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
from typing import NamedTuple

import torch

from . import capi
from .rotary_table import rotary_table


def _load_binding():
    path = os.path.join(os.path.dirname(capi.LIB_PATH), "_ttorch.so")
    if not os.path.exists(path):
        raise capi.NativeLibraryMissing(f"{path} not found. Build it with "
                                        f"`python {os.path.join(os.path.dirname(__file__), 'build.py')}`.")
    loader = importlib.machinery.ExtensionFileLoader("_ttorch", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_ttorch", loader))
    loader.exec_module(module)
    return module


_native = _load_binding()

_DT = {torch.float32: capi.TT_F32, torch.bfloat16: capi.TT_BF16}


def _done(result, explain, *args):
    """The result of a native call; None: an argument does not fit, int: the status of a call that failed."""
    if result is None:
        explain(*args)
        raise ValueError("arguments do not fit the call")
    capi.check(result)


def _check_inputs(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a torch.Tensor")
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D [B,H,rows,D], got shape {tuple(t.shape)}")
        if not t.is_cuda:
            raise ValueError(f"{name} is on {t.device}; attention runs on CUDA tensors only (no CPU path)")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k, v must share dtype float32 or bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    if k.shape[0] != B or Hkv < 1 or H % Hkv != 0 or k.shape[3] != D or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)} "
                         "(k, v heads must divide q heads)")
    return B, H, S, k.shape[2], D


def _stream_ptr(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _check_lens(kv_lens, B, device):
    if kv_lens is None:
        return None
    if not isinstance(kv_lens, torch.Tensor) or kv_lens.dtype != torch.int32 or not kv_lens.is_cuda \
            or not kv_lens.is_contiguous() or tuple(kv_lens.shape) != (B,):
        raise ValueError(f"kv_lens must be a contiguous CUDA int32 tensor of shape ({B},)")
    return kv_lens


def _explain_attention(q, k, v, kv_lens=None, out=None, lse=None, dout=None, decode=False):
    B, H, S, _, _ = _check_inputs(q, k, v)
    _check_lens(kv_lens, B, q.device)
    if decode and S != 1:
        raise ValueError(f"decode needs S == 1, got {S}")
    if dout is not None:
        for name, t, shp in (("out", out, q.shape), ("dout", dout, q.shape)):
            if tuple(t.shape) != tuple(shp) or t.dtype != q.dtype or not t.is_cuda or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous CUDA tensor of shape {tuple(shp)} and dtype {q.dtype}")
        if tuple(lse.shape) != (B, H, S) or lse.dtype != torch.float32 or not lse.is_cuda or not lse.is_contiguous():
            raise ValueError("lse must be contiguous CUDA float32 [B,H,S]")


def attention_forward(q, k, v, causal=False, scale=None, out=None, lse=None, need_lse=True, kv_lens=None):
    """`softmax(scale * q k^T [+causal]) v` -> (out, lse).  Asynchronous on the current stream.
    `kv_lens` (int32 `[B]`, CUDA): batch entry b attends to its first kv_lens[b] keys only."""
    r = _native.attention_forward(q, k, v, causal, scale, out, lse, need_lse, kv_lens)
    return r if r.__class__ is tuple else _done(r, _explain_attention, q, k, v, kv_lens)


def attention_backward(q, k, v, out, lse, dout, causal=False, scale=None, workspace=None, kv_lens=None):
    """(dq, dk, dv) for upstream gradient `dout`; `out`, `lse` from `attention_forward` (same `kv_lens`)."""
    r = _native.attention_backward(q, k, v, out, lse, dout, causal, scale, workspace, kv_lens)
    return r if r.__class__ is tuple else _done(r, _explain_attention, q, k, v, kv_lens, out, lse, dout)


def _explain_varlen(q, k, v, cu_q, cu_k):
    for name, t in (("q", q), ("k", k)):
        if t.dim() != 3 or not t.is_cuda or not t.is_contiguous() or t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be a contiguous CUDA bfloat16 tensor [tokens, heads, D]")
    for name, t in (("cu_q", cu_q), ("cu_k", cu_k)):
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.dim() != 1 or t.numel() != cu_q.numel():
            raise ValueError(f"{name} must be a contiguous CUDA int32 vector of n_seq + 1 cumulative token counts")
    if k.shape[2] != q.shape[2] or k.shape[1] < 1 or q.shape[1] % k.shape[1] != 0:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)}")
    raise ValueError("v, out, lse and dout must be CUDA tensors, max_q and max_k 32-bit integers")


def attention_forward_varlen(q, k, v, cu_q, cu_k, max_q, max_k, causal=False, scale=None, out=None, lse=None):
    """Packed variable-length batch: q `[total_q,H,D]`, k, v `[total_k,Hkv,D]`, cu_q / cu_k int32 `[n_seq+1]`
    (CUDA) cumulative token counts, max_q / max_k the longest sequence.  Returns (out `[total_q,H,D]`,
    lse `[H,total_q]`)."""
    r = _native.attention_forward_varlen(q, k, v, cu_q, cu_k, max_q, max_k, causal, scale, out, lse)
    return r if r.__class__ is tuple else _done(r, _explain_varlen, q, k, v, cu_q, cu_k)


def attention_backward_varlen(q, k, v, cu_q, cu_k, max_q, max_k, out, lse, dout, causal=False, scale=None, workspace=None):
    """(dq, dk, dv) of the packed batch; `out`, `lse` from `attention_forward_varlen`."""
    r = _native.attention_backward_varlen(q, k, v, cu_q, cu_k, max_q, max_k, out, lse, dout, causal, scale, workspace)
    return r if r.__class__ is tuple else _done(r, _explain_varlen, q, k, v, cu_q, cu_k)


def set_backward_deterministic(on: bool) -> None:
    """True: the tensor-core backward always runs its two-pass, bit-reproducible kernels; False: whichever
    measured faster for the shape, for larger problems the single-pass one, whose dq repeats to fp32 rounding
    only.  Never called: the two passes for packed batches and at head dim 128, as False at head dim 64.
    Process-wide."""
    capi.check(capi.lib.tt_attn_bwd_set_deterministic(1 if on else 0))


def decode_workspace_bytes(B, H, L, D, dtype=torch.bfloat16, Hkv=None) -> int:
    d = capi.make_desc(B, H, 1, L, D, _DT[dtype], False, None, Hkv=Hkv)
    return int(capi.lib.tt_attn_decode_workspace_bytes(ctypes.byref(d)))


def attention_decode(q, k, v, scale=None, out=None, lse=None, workspace=None, need_lse=True):
    """Single-query attention: q `[B,H,1,D]` against the whole cache k,v `[B,H,L,D]`."""
    r = _native.attention_decode(q, k, v, scale, out, lse, workspace, need_lse)
    return r if r.__class__ is tuple else _done(r, lambda: _explain_attention(q, k, v, decode=True))


def _explain_paged(q, k_pool, v_pool, block_table, seq_lens, max_len):
    if q.dim() != 4 or q.shape[2] != 1 or not q.is_cuda or not q.is_contiguous() or q.dtype != torch.bfloat16:
        raise ValueError("q must be a contiguous CUDA bfloat16 tensor [B,H,1,D]")
    B, H, _, D = q.shape
    for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
        if t.dim() != 4 or not t.is_cuda or not t.is_contiguous() or t.dtype != q.dtype or t.shape[3] != D:
            raise ValueError(f"{name} must be a contiguous CUDA bfloat16 tensor with last axis {D}")
    if tuple(k_pool.shape) != tuple(v_pool.shape):
        raise ValueError("k_pool and v_pool must have one shape")
    for name, t, shp in (("block_table", block_table, None), ("seq_lens", seq_lens, (B,))):
        if t is not None and (t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or
                              (shp is not None and tuple(t.shape) != shp)):
            raise ValueError(f"{name} must be a contiguous CUDA int32 tensor" + (f" of shape {shp}" if shp else ""))
    Hkv = k_pool.shape[1]
    if H % Hkv != 0:
        raise ValueError(f"key/value heads {Hkv} must divide query heads {H}")
    if block_table is not None:
        if block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError("block_table must be [B, max_pages]")
    else:
        if k_pool.shape[0] != B:
            raise ValueError("a dense cache must be [B,Hkv,L,D]")
        if max_len is not None and int(max_len) > k_pool.shape[2]:
            raise ValueError("max_len exceeds the cache length")
    raise ValueError("out, lse and workspace must be CUDA tensors, and lengths 32-bit integers")


def attention_decode_paged(q, k_pool, v_pool, block_table=None, seq_lens=None, max_len=None, scale=None, out=None,
                           lse=None, workspace=None, need_lse=True):
    """Single-query attention over a paged and/or ragged cache (bf16, D 64 or 128).

    q `[B,H,1,D]`.  With `block_table` (int32 `[B, max_pages]`, CUDA): k_pool, v_pool are page pools
    `[pages, Hkv, page_size, D]`.  Without: dense `[B,Hkv,L,D]`.  `seq_lens` (int32 `[B]`, CUDA)
    limits each batch entry to its first seq_lens[b] keys.  `max_len`: longest possible sequence
    (default: page_size * max_pages, or L of the dense cache)."""
    r = _native.attention_decode_paged(q, k_pool, v_pool, block_table, seq_lens, max_len, scale, out, lse, workspace, need_lse)
    return r if r.__class__ is tuple else _done(r, _explain_paged, q, k_pool, v_pool, block_table, seq_lens, max_len)


class CacheStep(NamedTuple):
    """What `cache_extend` says of the new tokens: lengths with them, pages left, cumulative counts `[B+1]`, and for
    each packed row its slot in the cache (-1 behind the last row) and its position."""
    seq_lens: torch.Tensor
    n_free: torch.Tensor
    cu_new: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


def _explain_tables(block_table, seq_lens, more, out=None, sizes=()):
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2 or block_table.dtype != torch.int32 \
            or not block_table.is_cuda or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous CUDA int32 tensor [B, max_pages]")
    B = block_table.shape[0]
    for name, t, n, types in [("seq_lens", seq_lens, B, (torch.int32,))] + more:
        if not isinstance(t, torch.Tensor) or t.dtype not in types or t.device != block_table.device \
                or not t.is_contiguous() or t.dim() != 1 or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name} must be a contiguous {types[0]} vector" + (f" of {n}" if n is not None else "") +
                             " on block_table's device")
    if out is not None:
        raise ValueError(f"out must be a tuple of contiguous int32 vectors of {sizes} elements on block_table's device")
    raise ValueError("page_size and max_tokens must be 32-bit integers, max_tokens not negative")


def cache_extend(block_table, seq_lens, new_lens, free_pages, n_free, page_size, max_tokens, out=None):
    """Pages and slots for `new_lens` more tokens of each request, on the GPU -> `CacheStep`.

    `block_table` `[B, max_pages]` gets the new pages' columns; `free_pages` with `n_free` `[1]` page numbers on it is used
    from its end and not written.  Requests are served in their order until one's tokens exceed `max_tokens` in all or its
    pages what is free; it and those behind it get nothing (their lengths stay).  All tensors int32, CUDA.  `out`: a
    `CacheStep` to write into; it must not share memory with the inputs, so a loop keeps two and takes them in turn."""
    r = _native.cache_extend(block_table, seq_lens, new_lens, free_pages, n_free, page_size, max_tokens, out)
    if r.__class__ is tuple:
        return tuple.__new__(CacheStep, r)
    i32 = (torch.int32,)
    return _done(r, lambda: _explain_tables(block_table, seq_lens, [
        ("new_lens", new_lens, block_table.shape[0], i32), ("free_pages", free_pages, None, i32), ("n_free", n_free, 1, i32)], out,
        "B, 1, B + 1, max_tokens, max_tokens"))


def cache_release(block_table, seq_lens, done, free_pages, n_free, page_size, out=None):
    """The pages of the requests that `done` (bool `[B]`) marks, back on `free_pages` behind its `n_free` -> (seq_lens with
    0 there, n_free).  Negative entries of their rows are no pages and are left out.  `out`: those two tensors, apart from the inputs."""
    r = _native.cache_release(block_table, seq_lens, done, free_pages, n_free, page_size, out)
    if r.__class__ is tuple:
        return r
    return _done(r, lambda: _explain_tables(block_table, seq_lens, [
        ("done", done, block_table.shape[0], (torch.bool, torch.uint8)), ("free_pages", free_pages, None, (torch.int32,)),
        ("n_free", n_free, 1, (torch.int32,))], out, "B, 1"))


def _page_bytes(bits, page_size, head_dim):
    call = capi.lib.tt_cache_q4_page_bytes if bits == 4 else capi.lib.tt_cache_q8_page_bytes
    return int(call(int(page_size), int(head_dim)))


def _page_tokens(bits, n_bytes, head_dim):
    """The page size whose pages have that many bytes; 0: none has."""
    if head_dim not in (64, 128):
        return 0
    lo, hi = 0, n_bytes // (8 * head_dim) + 1   # in units of 16
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if _page_bytes(bits, 16 * mid, head_dim) <= n_bytes else (lo, mid)
    return 16 * lo if lo and _page_bytes(bits, 16 * lo, head_dim) == n_bytes else 0


def _cache_alloc(bits, pages, kv_heads, page_size, head_dim, device):
    n = _page_bytes(bits, page_size, head_dim)
    if n == 0:
        raise ValueError(f"page_size {page_size} must be a multiple of 16 and head_dim {head_dim} 64 or 128")
    k = torch.zeros((int(pages), int(kv_heads), n), dtype=torch.uint8, device=device)
    return k, torch.zeros_like(k)


def cache_alloc_q4(pages, kv_heads, page_size, head_dim, device="cuda"):
    """(k_cache, v_cache) of a 4-bit key/value cache: zeroed bytes `[pages, kv_heads, page bytes]`, head dim 64 or 128, pages
    of a multiple of 16 tokens.  4.25 bits a value: per 32 channels a scale of 8 bits and 4 bits each."""
    return _cache_alloc(4, pages, kv_heads, page_size, head_dim, device)


def cache_alloc_q8(pages, kv_heads, page_size, head_dim, device="cuda"):
    """(k_cache, v_cache) of an 8-bit key/value cache, as `cache_alloc_q4`: 8-bit floats (e4m3) and for every 16 tokens of a head a scale, a power of two."""
    return _cache_alloc(8, pages, kv_heads, page_size, head_dim, device)


def _explain_cache(bits, k_cache, v_cache):
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.uint8 or t.dim() != 3 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous CUDA uint8 tensor [pages, kv_heads, page bytes], see cache_alloc_q{bits}")
    if k_cache.shape != v_cache.shape or k_cache.device != v_cache.device:
        raise ValueError("k_cache and v_cache must have one shape and device")


def _explain_cache_append(bits, k, v, slots, k_cache, v_cache):
    _explain_cache(bits, k_cache, v_cache)
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dtype not in _DT or t.device != k_cache.device or t.dim() != 3 or t.stride(2) != 1:
            raise ValueError(f"{name} must be a float32/bfloat16 tensor [T, kv_heads, D] on the cache's device, channels next to each other")
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must have one shape and type")
    if k.shape[1] != k_cache.shape[1]:
        raise ValueError(f"k has {k.shape[1]} heads, the cache {k_cache.shape[1]}")
    if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int32 or slots.device != k_cache.device or tuple(slots.shape) != (k.shape[0],) \
            or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int32 vector of {k.shape[0]} on the cache's device")
    raise ValueError(f"pages of {k_cache.shape[2]} bytes are not a multiple of 16 tokens of head dim {k.shape[2]} (64 or 128)")


def cache_append_q4(k, v, slots, k_cache, v_cache):
    """New keys and values `[T, kv_heads, D]` (float32 or bfloat16, strided) into a 4-bit cache at `slots` (int32 `[T]`, as from
    `cache_extend`; -1 is passed over, no slot may come twice) -> (k_cache, v_cache), written in place."""
    r = _native.cache_append_q4(k, v, slots, k_cache, v_cache)
    return r if r.__class__ is tuple else _done(r, _explain_cache_append, 4, k, v, slots, k_cache, v_cache)


def cache_append_q8(k, v, slots, k_cache, v_cache):
    """New keys and values into an 8-bit cache, as `cache_append_q4`.  The tokens of a call that go to one block of 16 rows of a page lie next to each
    other and each has a slot of its own, as a sequence's do (else that block is unspecified).  A block's scale is the smallest power of two that holds its tokens' largest value; tokens that come later raise
    it where they have to, and a call that brings the block's first row begins it anew."""
    r = _native.cache_append_q8(k, v, slots, k_cache, v_cache)
    return r if r.__class__ is tuple else _done(r, _explain_cache_append, 8, k, v, slots, k_cache, v_cache)


def _explain_cache_read(bits, k_cache, v_cache, block_table, cu_lens, total, page_size):
    _explain_cache(bits, k_cache, v_cache)
    dev = k_cache.device
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32 or block_table.device != dev or block_table.dim() != 2 \
            or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 tensor [B, max_pages] on the cache's device")
    n = block_table.shape[0] + 1
    if not isinstance(cu_lens, torch.Tensor) or cu_lens.dtype != torch.int32 or cu_lens.device != dev or tuple(cu_lens.shape) != (n,) \
            or not cu_lens.is_contiguous():
        raise ValueError(f"cu_lens must be a contiguous int32 vector of {n} cumulative token counts on the cache's device")
    if int(page_size) < 16 or int(page_size) % 16 or int(page_size) not in [_page_tokens(bits, k_cache.shape[2], d) for d in (64, 128)]:
        raise ValueError(f"pages of {k_cache.shape[2]} bytes are not {page_size} tokens (a multiple of 16) of head dim 64 or 128")
    raise ValueError("total must be a 32-bit integer, k and v contiguous bfloat16 [total, kv_heads, D] on the cache's device")


def cache_read_q4(k_cache, v_cache, block_table, cu_lens, total, page_size, k=None, v=None):
    """The first `cu_lens[b+1] - cu_lens[b]` tokens of each sequence of a 4-bit cache as packed bfloat16 k, v `[total, kv_heads, D]`:
    the keys of `attention_forward_varlen` with `cu_k = cu_lens`, for prompt tokens that follow what is cached.  Rows of given
    `k`, `v` from `cu_lens[B]` on stay as they are."""
    r = _native.cache_read_q4(k_cache, v_cache, block_table, cu_lens, total, page_size, k, v)
    return r if r.__class__ is tuple else _done(r, _explain_cache_read, 4, k_cache, v_cache, block_table, cu_lens, total, page_size)


def cache_read_q8(k_cache, v_cache, block_table, cu_lens, total, page_size, k=None, v=None):
    """The tokens of an 8-bit cache's sequences as packed bfloat16, as `cache_read_q4`."""
    r = _native.cache_read_q8(k_cache, v_cache, block_table, cu_lens, total, page_size, k, v)
    return r if r.__class__ is tuple else _done(r, _explain_cache_read, 8, k_cache, v_cache, block_table, cu_lens, total, page_size)


def _explain_cache_decode(bits, q, k_cache, v_cache, block_table, seq_lens, max_len, out, lse):
    _explain_cache(bits, k_cache, v_cache)
    dev = k_cache.device
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[2] != 1 or q.dtype != torch.bfloat16 or q.device != dev or not q.is_contiguous():
        raise ValueError("q must be a contiguous bfloat16 tensor [B,H,1,D] on the cache's device")
    B, H, _, D = q.shape
    Hkv = k_cache.shape[1]
    if Hkv < 1 or H % Hkv != 0:
        raise ValueError(f"key/value heads {Hkv} must divide query heads {H}")
    page = _page_tokens(bits, k_cache.shape[2], D)
    if page == 0:
        raise ValueError(f"pages of {k_cache.shape[2]} bytes are not a multiple of 16 tokens of head dim {D} (64 or 128)")
    for name, t, shape in (("block_table", block_table, None), ("seq_lens", seq_lens, (B,))):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != dev or not t.is_contiguous()
                              or (shape is not None and tuple(t.shape) != shape)):
            raise ValueError(f"{name} must be a contiguous int32 tensor on the cache's device" + (f" of shape {shape}" if shape else ""))
    if block_table is not None and (block_table.dim() != 2 or block_table.shape[0] != B):
        raise ValueError("block_table must be [B, max_pages]")
    if block_table is None and k_cache.shape[0] != B:
        raise ValueError("a cache without a block table must have one page per batch entry")
    longest = page * (1 if block_table is None else block_table.shape[1])
    if max_len is not None and int(max_len) > longest:
        raise ValueError(f"max_len exceeds the {longest} keys that a sequence may have")
    for name, t, shape, dtype in (("out", out, q.shape, torch.bfloat16), ("lse", lse, (B, H, 1), torch.float32)):
        if t is not None and (not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape) or t.dtype != dtype or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on the cache's device")
    raise ValueError("workspace must be a contiguous tensor on the cache's device, and lengths 32-bit integers")


def attention_decode_q4(q, k_cache, v_cache, block_table=None, seq_lens=None, max_len=None, scale=None, out=None, lse=None, workspace=None, need_lse=True):
    """Single-query attention over a 4-bit cache (see `cache_alloc_q4`) -> (out, lse), as `attention_decode_paged` over a 16-bit one.

    q `[B,H,1,D]` bfloat16, D 64 or 128.  `block_table` (int32 `[B, max_pages]`) names each sequence's pages; None: batch entry b has
    page b to itself.  `seq_lens` (int32 `[B]`): keys of each sequence.  `max_len`: longest possible sequence (default: what the pages
    can hold), which decides how the keys are divided.  An empty sequence gives out = 0, lse = -inf.  A group of more than 16 query heads reads the
    cache once for each 16."""
    r = _native.attention_decode_q4(q, k_cache, v_cache, block_table, seq_lens, max_len, scale, out, lse, workspace, need_lse)
    return r if r.__class__ is tuple else _done(r, _explain_cache_decode, 4, q, k_cache, v_cache, block_table, seq_lens, max_len, out, lse)


def attention_decode_q8(q, k_cache, v_cache, block_table=None, seq_lens=None, max_len=None, scale=None, out=None, lse=None, workspace=None, need_lse=True):
    """Single-query attention over an 8-bit cache (see `cache_alloc_q8`) -> (out, lse), with the arguments of `attention_decode_q4`."""
    r = _native.attention_decode_q8(q, k_cache, v_cache, block_table, seq_lens, max_len, scale, out, lse, workspace, need_lse)
    return r if r.__class__ is tuple else _done(r, _explain_cache_decode, 8, q, k_cache, v_cache, block_table, seq_lens, max_len, out, lse)


def rotary_frequencies(rotary_dim, base=10000.0, sections=None, cyclic=False, own_ladder=False, device="cuda"):
    """(inv_freq `[rotary_dim/2]` float64, axes int32 or None) of `rotary_forward`.

    `sections`: the pairs of each axis, `rotary_dim / 2` in all (None: one axis).  Pairs go to the axes section by section, or
    with `cyclic` in turn, as long as an axis has some left.  Pair i of n turns by `base ** (-i / n)` per position;
    with `own_ladder` each axis counts its own pairs, i.e. it has slow and fast ones as an axis alone would."""
    freq, axes, n_axes = rotary_table(rotary_dim, base, sections, cyclic, own_ladder)
    return (torch.tensor(freq, dtype=torch.float64, device=device),
            torch.tensor(axes, dtype=torch.int32, device=device) if n_axes > 1 else None)


def _explain_rotary(q, k, positions, inv_freq, axes, out_q, out_k):
    for name, t in (("q", q), ("k", k), ("out_q", out_q), ("out_k", out_k)):
        if t is None and name != "q":
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DT or t.dim() not in (3, 4) \
                or (t.shape[-1] > 1 and t.stride(-1) != 1):
            raise ValueError(f"{name} must be a CUDA float32/bfloat16 tensor [T,H,D] or [B,H,S,D] whose channels lie next to each other")
        if t.dtype != q.dtype or t.dim() != q.dim() or t.device != q.device:
            raise ValueError(f"{name} must have q's type, dimensions and device")
    for name, t, x in (("out_q", out_q, q), ("out_k", out_k, k)):
        if t is not None and (x is None or t.shape != x.shape):
            raise ValueError(f"{name} must have its input's shape")
    rows = 0 if q.dim() == 3 else 2
    if k is not None and (k.shape[rows] != q.shape[rows] or k.shape[-1] != q.shape[-1] or (rows and k.shape[0] != q.shape[0])):
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} k {tuple(k.shape)}")
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.device != q.device \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 vector on q's device, one frequency per pair")
    if axes is not None and (not isinstance(axes, torch.Tensor) or axes.dtype != torch.int32 or axes.shape != inv_freq.shape
                             or axes.device != q.device or not axes.is_contiguous()):
        raise ValueError("axes must be a contiguous int32 vector on q's device, one axis per pair")
    if axes is None and isinstance(positions, torch.Tensor) and positions.dim() > 1 and positions.shape[0] != 1:
        raise ValueError(f"positions {tuple(positions.shape)} are of {positions.shape[0]} axes, without `axes` there is one: [1, B, S] for positions of each batch entry")
    want = "[axes, T] or [T]" if q.dim() == 3 else "[axes, B, S], [axes, S] or [S]"
    raise ValueError(f"positions must be an int32 tensor {want} on q's device, rows next to each other")


def rotary_forward(q, k, positions, inv_freq, axes=None, interleaved=False, scale=None, out_q=None, out_k=None):
    """Query and key heads turned by their positions -> (q, k), inputs `[T,H,D]` (packed) or `[B,H,S,D]`, k may be None.

    Pair i of the first `2 * len(inv_freq)` channels turns by `positions[axes[i]] * inv_freq[i]` (float64 `[R/2]`, int32 `[R/2]` or
    None, see `rotary_frequencies`): channels i and i + R/2, or with `interleaved` 2i and 2i + 1; the other channels are copied.
    positions: int32 `[axes, T]` / `[axes, B, S]` / `[axes, S]`, or `[T]` / `[S]` with one axis; without `axes` there is one, and more
    rows are refused (position ids `[B, S]` are `[1, B, S]` here).  Strided inputs are fine as long
    as channels lie next to each other; `out_q`, `out_k` may be the inputs themselves.  `scale` (1) multiplies the channels that turn."""
    r = _native.rotary(q, k, positions, inv_freq, axes, interleaved, scale, False, out_q, out_k)
    return r if r.__class__ is tuple else _done(r, _explain_rotary, q, k, positions, inv_freq, axes, out_q, out_k)


def rotary_backward(dq, dk, positions, inv_freq, axes=None, interleaved=False, scale=None, out_q=None, out_k=None):
    """(dq, dk) with respect to the inputs of `rotary_forward` for upstream gradients `dq`, `dk` of its results."""
    r = _native.rotary(dq, dk, positions, inv_freq, axes, interleaved, scale, True, out_q, out_k)
    return r if r.__class__ is tuple else _done(r, _explain_rotary, dq, dk, positions, inv_freq, axes, out_q, out_k)


def _explain_weights(x, pairs):
    seen = None
    for name, w, wanted in pairs:
        if not wanted and w is not None:
            raise ValueError(f"{name} goes with the heads it weights")
        if wanted and (not isinstance(w, torch.Tensor) or w.dtype not in (x.dtype, torch.float32) or w.device != x.device or tuple(w.shape) != (x.shape[-1],)
                       or not w.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous vector of {x.shape[-1]}, float32 or of the heads' type, on the heads' device")
        if wanted and seen is not None and w.dtype != seen:
            raise ValueError("q_weight and k_weight must have one type")
        seen = w.dtype if wanted else seen


def _explain_norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, axes, out_q, out_k, x=()):
    if not isinstance(q, torch.Tensor):
        raise ValueError("q must be a CUDA float32/bfloat16 tensor [T,H,D] or [B,H,S,D]")
    for name, t, g in x:
        if (t is None) != (g is None) or (t is not None and (not isinstance(t, torch.Tensor) or not isinstance(g, torch.Tensor) or t.shape != g.shape
                                                            or t.dtype != g.dtype or t.device != g.device or (t.shape[-1] > 1 and t.stride(-1) != 1))):
            raise ValueError(f"{name} must have its gradient's shape, type and device, channels next to each other")
    _explain_weights(q, (("q_weight", q_weight, True), ("k_weight", k_weight, k is not None)))
    _explain_rotary(q, k, positions, inv_freq, axes, out_q, out_k)


def norm_rotary_forward(q, k, q_weight, k_weight, positions, inv_freq, axes=None, interleaved=False, eps=1e-6, scale=None, out_q=None, out_k=None):
    """Query and key heads normed and turned by their positions in one pass -> (q, k); k (with its weight) may be None.

    Each head is divided by the root of its channels' mean square and `eps`, multiplied by a weight per channel (`[D]`, float32 or of
    the heads' type) and turned as by `rotary_forward`, whose arguments the others are."""
    r = _native.norm_rotary_forward(q, k, q_weight, k_weight, positions, inv_freq, axes, interleaved, eps, scale, out_q, out_k)
    return r if r.__class__ is tuple else _done(r, _explain_norm_rotary, q, k, q_weight, k_weight, positions, inv_freq, axes, out_q, out_k)


def norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, axes=None, interleaved=False, eps=1e-6, scale=None, out_q=None,
                         out_k=None, workspace=None):
    """(dq, dk, dq_weight, dk_weight) of `norm_rotary_forward` on q, k for upstream gradients `dq`, `dk` of its results.  `out_q`, `out_k` may be
    `dq`, `dk` themselves."""
    r = _native.norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, axes, interleaved, eps, scale, out_q, out_k, workspace)
    return r if r.__class__ is tuple else _done(r, _explain_norm_rotary, dq, dk, q_weight, k_weight, positions, inv_freq, axes, out_q, out_k,
                                                (("q", q, dq), ("k", k, dk)))


def _explain_append_rotary(q, k, v, slots, positions, inv_freq, k_pool, v_pool, axes, q_weight, k_weight, out_q, out_k):
    for name, t in (("k", k), ("q", q), ("v", v)):
        if t is None and name == "q":
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DT or t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
            raise ValueError(f"{name} must be a CUDA float32/bfloat16 tensor [T, heads, D] whose channels lie next to each other")
        if t.dtype != k.dtype or t.device != k.device or t.shape[0] != k.shape[0] or t.shape[2] != k.shape[2]:
            raise ValueError(f"{name} must have k's type, device, tokens and head dim")
    if v.shape != k.shape:
        raise ValueError(f"shape mismatch: k {tuple(k.shape)} v {tuple(v.shape)}")
    if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int32 or slots.device != k.device or tuple(slots.shape) != (k.shape[0],) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int32 vector of {k.shape[0]} on k's device")
    for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.device != k.device or t.dim() != 4 or not t.is_contiguous() \
                or t.shape[1] != k.shape[1] or t.shape[3] != k.shape[2] or t.shape != k_pool.shape:
            raise ValueError(f"{name} must be a contiguous bfloat16 tensor [pages, {k.shape[1]}, page_size, {k.shape[2]}] on k's device")
    for name, t, x in (("out_q", out_q, q), ("out_k", out_k, k)):
        if t is not None and (x is None or not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.shape != x.shape or t.device != k.device
                              or (t.shape[2] > 1 and t.stride(2) != 1)):
            raise ValueError(f"{name} must be a bfloat16 tensor of its input's shape and device")
    _explain_weights(k, (("q_weight", q_weight, q is not None and k_weight is not None), ("k_weight", k_weight, k_weight is not None)))
    _explain_rotary(k, None, positions, inv_freq, axes, None, None)


def cache_append_rotary(q, k, v, slots, positions, inv_freq, k_pool, v_pool, axes=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6,
                        scale=None, out_q=None, out_k=None):
    """A step's tokens on their way to `attention_decode_paged`: q turned by its positions -> bfloat16 `[T, H, D]`, and keys (turned) and values
    written into their slots of the bfloat16 pools `[pages, kv_heads, page_size, D]`, D 64 or 128.

    q `[T, H, D]` (or None), k, v `[T, kv_heads, D]`, float32 or bfloat16, strided; `slots`, `positions` as from `cache_extend`; a slot of -1 is passed
    over, and none may come twice.  With `q_weight` and `k_weight` heads are normed first, as by `norm_rotary_forward`.  `out_k`: a bfloat16 tensor of k's
    shape that gets the turned keys too, for attention over the new tokens themselves.  `scale` multiplies the channels that turn."""
    r = _native.cache_append_rotary(q, k, v, slots, positions, inv_freq, k_pool, v_pool, axes, interleaved, q_weight, k_weight, eps, scale, out_q, out_k)
    return r[0] if r.__class__ is tuple else _done(r, _explain_append_rotary, q, k, v, slots, positions, inv_freq, k_pool, v_pool, axes, q_weight, k_weight, out_q, out_k)


def _explain_softmax_forward(x):
    raise ValueError("softmax_forward takes a contiguous float32/bfloat16 CUDA tensor")


def softmax_forward(x, out=None):
    """Softmax over the last axis of a contiguous CUDA tensor (float32 or bfloat16)."""
    r = _native.softmax_forward(x, out)
    return r if r is not None and r.__class__ is not int else _done(r, _explain_softmax_forward, x)


def _explain_softmax_backward(y, dy):
    raise ValueError("softmax_backward takes two contiguous CUDA tensors of one shape and dtype")


def softmax_backward(y, dy, dx=None):
    """dx = y * (dy - sum(dy * y, last axis)) for y = softmax(x)."""
    r = _native.softmax_backward(y, dy, dx)
    return r if r is not None and r.__class__ is not int else _done(r, _explain_softmax_backward, y, dy)


def _explain_fc(x, w, bias=None, dy=None):
    if not (x.is_cuda and w.is_cuda and x.is_contiguous() and w.is_contiguous()) or x.dtype != w.dtype \
            or x.dtype not in _DT or w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[0]:
        raise ValueError("fc takes contiguous CUDA tensors x [..., in] and w [in, out] of one dtype (float32/bfloat16)")
    if dy is not None:
        raise ValueError("dy must be a contiguous CUDA tensor shaped like the layer's output")
    raise ValueError(f"bias must be a CUDA tensor of shape ({w.shape[1]},) and dtype {x.dtype}")


def fc_forward(x, w, bias=None, out=None):
    """y = x @ w + bias for x `[..., in]`, w `[in, out]`, bias `[out]` or None."""
    r = _native.fc_forward(x, w, bias, out)
    return r if r is not None and r.__class__ is not int else _done(r, _explain_fc, x, w, bias)


def fc_backward(x, w, dy, need_dx=True, need_dw=True, need_db=True, scalar_bias=False, workspace=None):
    """(dx, dw, db) of `fc_forward` for upstream gradient dy `[..., out]`; skipped ones are None."""
    r = _native.fc_backward(x, w, dy, need_dx, need_dw, need_db, scalar_bias, workspace)
    return r if r.__class__ is tuple else _done(r, _explain_fc, x, w, None, dy)


def check_device_status(device=None):
    """Synchronises the current stream and raises if a bounded device-side wait expired."""
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        capi.check(capi.lib.tt_check_device_status(st))


# ------------------------------------------------------------------ host-buffer calls
def _host_ptr(t):
    if t is None:
        return None
    if t.is_cuda or not t.is_contiguous():
        raise ValueError("host-buffer calls take contiguous CPU tensors")
    return ctypes.c_void_p(t.data_ptr())


def attention_forward_host(q, k, v, causal=False, scale=None, out=None, lse=None):
    """Same as `attention_forward` for CPU (ideally pinned) tensors: upload, run, download."""
    B, H, S, D = q.shape
    L = k.shape[2]
    if out is None:
        out = torch.empty_like(q)
    if lse is None:
        lse = torch.empty((B, H, S), dtype=torch.float32)
    d = capi.make_desc(B, H, S, L, D, _DT[q.dtype], causal, scale, Hkv=k.shape[1])
    capi.check(capi.lib.tt_attn_fwd_host(ctypes.byref(d), _host_ptr(q), _host_ptr(k), _host_ptr(v),
                                         _host_ptr(out), _host_ptr(lse)))
    return out, lse


def attention_backward_host(q, k, v, out, lse, dout, causal=False, scale=None, dq=None, dk=None, dv=None):
    B, H, S, D = q.shape
    L = k.shape[2]
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    d = capi.make_desc(B, H, S, L, D, _DT[q.dtype], causal, scale, Hkv=k.shape[1])
    capi.check(capi.lib.tt_attn_bwd_host(ctypes.byref(d), _host_ptr(q), _host_ptr(k), _host_ptr(v), _host_ptr(out),
                                         _host_ptr(lse), _host_ptr(dout), _host_ptr(dq), _host_ptr(dk), _host_ptr(dv)))
    return dq, dk, dv


def attention_step_host(q, k, v, dout, causal=False, scale=None, out=None, lse=None, dq=None, dk=None, dv=None):
    """Forward + backward from CPU (pinned) tensors with uploads, kernels and downloads pipelined
    over slice chunks.  Returns (out, lse, dq, dk, dv)."""
    B, H, S, D = q.shape
    L = k.shape[2]
    out = torch.empty_like(q) if out is None else out
    lse = torch.empty((B, H, S), dtype=torch.float32) if lse is None else lse
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    d = capi.make_desc(B, H, S, L, D, _DT[q.dtype], causal, scale, Hkv=k.shape[1])
    capi.check(capi.lib.tt_attn_fwd_bwd_host(ctypes.byref(d), _host_ptr(q), _host_ptr(k), _host_ptr(v), _host_ptr(dout),
                                             _host_ptr(out), _host_ptr(lse), _host_ptr(dq), _host_ptr(dk), _host_ptr(dv)))
    return out, lse, dq, dk, dv


def attention_decode_host(q, k, v, scale=None, out=None, lse=None):
    B, H, S, D = q.shape
    L = k.shape[2]
    if out is None:
        out = torch.empty_like(q)
    if lse is None:
        lse = torch.empty((B, H, 1), dtype=torch.float32)
    d = capi.make_desc(B, H, 1, L, D, _DT[q.dtype], False, scale, Hkv=k.shape[1])
    capi.check(capi.lib.tt_attn_decode_host(ctypes.byref(d), _host_ptr(q), _host_ptr(k), _host_ptr(v),
                                            _host_ptr(out), _host_ptr(lse)))
    return out, lse
