"""Argument checks of the page-table and rotary calls (status codes, no GPU needed) and the frequency table."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")


def _buffers(n=8, size=4096):
    raw = (ctypes.c_char * (n * size))()
    base = ctypes.addressof(raw)
    base += -base % 256
    return raw, [ctypes.c_void_p(base + i * size) for i in range(n - 1)]


def _extend(tt, **kw):
    raw, p = _buffers(12)
    a = dict(table=p[0], lens=p[1], new=p[2], free=p[3], n_free=p[4], B=4, page=16, max_pages=8, cap=10, tokens=20, lens_out=p[5], n_free_out=p[6], cu=p[7],
             slots=p[8], pos=p[9])
    a.update({k: (p[v] if isinstance(v, str) and k else v) for k, v in kw.items()})
    rc = tt.capi.lib.tt_cache_extend(a["table"], a["lens"], a["new"], a["free"], a["n_free"], a["B"], a["page"], a["max_pages"], a["cap"], a["tokens"],
                                     a["lens_out"], a["n_free_out"], a["cu"], a["slots"], a["pos"], None)
    del raw
    return rc


def _at(p, offset):
    return ctypes.c_void_p(p.value + offset)


def test_extend_refuses_what_does_not_fit(tt):
    c = tt.capi
    for bad in (dict(B=0), dict(B=16385), dict(page=0), dict(max_pages=0), dict(cap=-1), dict(tokens=-1)):
        assert _extend(tt, **bad) == c.TT_ERR_BAD_SHAPE, bad
    for null in ("table", "lens", "new", "free", "n_free", "lens_out", "n_free_out", "cu", "slots", "pos"):
        assert _extend(tt, **{null: None}) == c.TT_ERR_NULL, null


def test_extend_and_release_refuse_outputs_on_inputs(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, p = _buffers(12)
    table, lens, new, free, n_free, lens_out, n_out, cu, slots, pos = p[:10]

    def extend(**kw):
        a = dict(table=table, lens=lens, new=new, free=free, n_free=n_free, lens_out=lens_out, n_out=n_out, cu=cu, slots=slots, pos=pos)
        a.update(kw)
        return lib.tt_cache_extend(a["table"], a["lens"], a["new"], a["free"], a["n_free"], 4, 16, 8, 10, 20, a["lens_out"], a["n_out"], a["cu"], a["slots"],
                                   a["pos"], None)

    for kw in (dict(lens_out=lens), dict(lens_out=_at(lens, 12)), dict(n_out=n_free), dict(cu=_at(new, -4)), dict(slots=pos), dict(pos=_at(free, 36)),
               dict(lens_out=_at(table, 124)), dict(n_out=_at(cu, 16))):
        assert extend(**kw) == c.TT_ERR_BAD_SHAPE and "overlaps" in c.last_error(), kw

    def release(**kw):
        a = dict(table=table, lens=lens, done=new, free=free, n_free=n_free, lens_out=lens_out, n_out=n_out)
        a.update(kw)
        return lib.tt_cache_release(a["table"], a["lens"], a["done"], a["free"], a["n_free"], a.get("B", 4), 16, 8, 10, a["lens_out"], a["n_out"], None)

    assert release(B=0) == c.TT_ERR_BAD_SHAPE and release(B=16385) == c.TT_ERR_BAD_SHAPE
    for null in ("table", "lens", "done", "free", "n_free", "lens_out", "n_out"):
        assert release(**{null: None}) == c.TT_ERR_NULL, null
    for kw in (dict(lens_out=lens), dict(n_out=n_free), dict(lens_out=free), dict(free=_at(table, 64)), dict(n_out=_at(lens_out, 12))):
        assert release(**kw) == c.TT_ERR_BAD_SHAPE and "overlaps" in c.last_error(), kw
    if not torch.cuda.is_available():
        assert extend() == c.TT_ERR_BAD_DEVICE and release() == c.TT_ERR_BAD_DEVICE
    del raw


def _rotary_desc(tt, **kw):
    d = tt.capi.RotaryDesc(B=2, S=4, H=4, Hkv=2, D=16, R=8, n_axes=1, dtype=tt.capi.TT_F32, interleaved=0, scale=1.0)
    d.q_stride[:] = d.q_out_stride[:] = (4 * 4 * 16, 4 * 16, 16)
    d.k_stride[:] = d.k_out_stride[:] = (2 * 4 * 16, 4 * 16, 16)
    d.pos_stride[:] = (8, 4)
    for name, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, name)[:] = v
        else:
            setattr(d, name, v)
    return d


def test_rotary_refuses_what_does_not_fit(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, p = _buffers(8)
    q, k, q_out, k_out, pos, freq = p[:6]

    def call(d, q=q, k=k, pos=pos, freq=freq, q_out=q_out, k_out=k_out):
        return lib.tt_rotary(ctypes.byref(d), q, k, pos, freq, None, 0, q_out, k_out, None)

    assert lib.tt_rotary(None, q, k, pos, freq, None, 0, q_out, k_out, None) == c.TT_ERR_NULL
    for bad in (dict(H=0), dict(Hkv=0), dict(D=1), dict(D=257), dict(R=0), dict(R=7), dict(R=18), dict(n_axes=0), dict(B=-1), dict(S=-1),
                dict(scale=math.inf), dict(scale=math.nan), dict(B=1 << 16, S=1 << 15), dict(q_stride=(-1, 64, 16)), dict(pos_stride=(-1, 4))):
        assert call(_rotary_desc(tt, **bad)) == c.TT_ERR_BAD_SHAPE, bad
    assert call(_rotary_desc(tt, dtype=7)) == c.TT_ERR_BAD_DTYPE
    # rows of an output that lie on each other
    for st in ((0, 64, 16), (256, 0, 16), (256, 64, 15), (64, 64, 16), (63, 256, 16)):
        assert call(_rotary_desc(tt, q_out_stride=st)) == c.TT_ERR_BAD_SHAPE, st
    d = _rotary_desc(tt)
    for kw in (dict(q=None), dict(q_out=None), dict(pos=None), dict(freq=None), dict(k=None), dict(k_out=None)):
        assert call(d, **kw) == c.TT_ERR_NULL, kw
    for kw in (dict(q_out=k), dict(q_out=_at(q, 64)), dict(k_out=_at(q, 512)), dict(k_out=q_out), dict(k_out=_at(q_out, 128)), dict(q_out=_at(k, 960)),
               dict(q=_at(q, 2))):
        assert call(d, **kw) == c.TT_ERR_BAD_SHAPE, kw
    assert call(_rotary_desc(tt, q_stride=(16, 32, 128)), q_out=q) == c.TT_ERR_BAD_SHAPE   # in place at other strides
    for empty in (dict(B=0), dict(S=0)):
        assert call(_rotary_desc(tt, **empty), q=None, pos=None) == c.TT_OK
    if not torch.cuda.is_available():
        assert call(d) == c.TT_ERR_BAD_DEVICE and call(d, q_out=q, k_out=k) == c.TT_ERR_BAD_DEVICE
    del raw


def _elements(at, st, n, D):
    import numpy as np
    i = np.indices(n).reshape(3, -1)
    return set(((at + (i * np.array(st)[:, None]).sum(0))[:, None] + np.arange(D)).reshape(-1).tolist())


@pytest.mark.parametrize("seed", range(4))
def test_rotary_outputs_among_the_rows_of_one_buffer(tt, seed):
    """Slices of one buffer at the same strides, shifted by rows, heads and odd numbers of elements: refused where they share an element, and only there."""
    import random
    if torch.cuda.is_available():
        pytest.skip("the accepted ones would run")
    lib, c, rng = tt.capi.lib, tt.capi, random.Random(seed)
    raw, (base,) = _buffers(2, 1 << 16)
    seen = {True: 0, False: 0}
    for _ in range(400):
        D, H, S, B, Hkv = rng.choice([2, 6, 16]), rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 3), rng.randint(1, 3)
        width = H + rng.randint(0, 6)
        st = [(width * S * D, D, width * D), (width * S * D, S * D, D), (D, S * B * D, B * D)][rng.randrange(3)]
        places = [rng.randrange(0, 8) * D + rng.choice([0, 0, 0, 1, -1]) + 8 for _ in range(2)] + [rng.choice([8, 8 + 4 * D, 8 + S * D]) + 4096 for _ in range(2)]
        d = _rotary_desc(tt, B=B, H=H, Hkv=Hkv, S=S, D=D, R=2, q_stride=st, q_out_stride=st, k_stride=st, k_out_stride=st)
        n = ((B, H, S), (B, Hkv, S))
        q, q_out, k, k_out = [_elements(at, st, n[i // 2], D) for i, at in enumerate(places)]
        meet = bool((q & q_out and places[0] != places[1]) or (k & k_out and places[2] != places[3]) or q & k_out or k & q_out or q_out & k_out)
        apart = all(len(e) == B * h * S * D for e, h in ((q_out, H), (k_out, Hkv)))
        rc = lib.tt_rotary(ctypes.byref(d), *[_at(base, 4 * at) for at in (places[0], places[2])], _at(base, 60000), _at(base, 60000), None, 0,
                           *[_at(base, 4 * at) for at in (places[1], places[3])], None)
        if apart:
            assert rc == (c.TT_ERR_BAD_SHAPE if meet else c.TT_ERR_BAD_DEVICE), (st, places, n, c.last_error())
            seen[meet] += 1
        else:
            assert rc == c.TT_ERR_BAD_SHAPE
    assert min(seen.values()) > 40
    # at strides of their own: refused where what they span overlaps
    d = _rotary_desc(tt, q_out_stride=(4 * 4 * 32, 4 * 32, 32))
    assert lib.tt_rotary(ctypes.byref(d), base, None, _at(base, 60000), _at(base, 60000), None, 0, _at(base, 4 * 64), None, None) == c.TT_ERR_BAD_SHAPE
    assert lib.tt_rotary(ctypes.byref(d), base, None, _at(base, 60000), _at(base, 60000), None, 0, _at(base, 4 * 512), None, None) == c.TT_ERR_BAD_DEVICE
    del raw


def test_calls_on_cpu_tensors_are_refused(tt):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="block_table"):
        tt.cache_extend(torch.zeros(4, 8, dtype=torch.int32), i, i, i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="block_table"):
        tt.cache_release(torch.zeros(4, 8, dtype=torch.int32), i, i.bool(), i, i[:1], 16)
    freq, _ = tt.rotary_frequencies(8, device="cpu")
    with pytest.raises(ValueError, match="q must be a CUDA"):
        tt.rotary_forward(torch.zeros(4, 2, 8), None, i, freq)


def test_frequencies(tt):
    freq, axes = tt.rotary_frequencies(8, base=100.0, device="cpu")
    assert axes is None and freq.dtype == torch.float64
    assert torch.allclose(freq, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15, atol=0)
    freq, axes = tt.rotary_frequencies(12, sections=(1, 3, 2), device="cpu")
    assert axes.tolist() == [0, 1, 1, 1, 2, 2]
    freq, axes = tt.rotary_frequencies(12, sections=(1, 3, 2), cyclic=True, device="cpu")
    assert axes.tolist() == [0, 1, 2, 1, 2, 1] and freq[1] == 10000.0 ** (-1 / 6)
    freq, axes = tt.rotary_frequencies(12, sections=(2, 0, 4), own_ladder=True, device="cpu")
    assert axes.tolist() == [0, 0, 2, 2, 2, 2] and freq.tolist() == [10000.0 ** -(i / n) for n in (2, 4) for i in range(n)]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, sections=(1, 2)), dict(rotary_dim=8, sections=(5, -1)), dict(rotary_dim=8, base=0.0)):
        with pytest.raises(ValueError):
            tt.rotary_frequencies(**bad, device="cpu")


def test_q4_cache_refuses_what_does_not_fit(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, p = _buffers(10, 1 << 16)
    k, v, slots, kc, vc, table, cu, ok, ov = p[:9]
    st = (ctypes.c_int64 * 2)(128, 64)
    assert [lib.tt_cache_q4_page_bytes(*a) for a in ((16, 64), (48, 128), (8, 64), (24, 64), (16, 96), (0, 64), (-16, 128))] == [16 * 34, 48 * 68, 0, 0, 0, 0, 0]

    def append(k=k, v=v, slots=slots, T=4, hkv=2, D=64, dtype=0, ks=st, vs=st, kc=kc, vc=vc, pages=3, page=16):
        return lib.tt_cache_append_q4(k, v, slots, T, hkv, D, dtype, ks, vs, kc, vc, pages, page, None)

    assert append(D=96) == c.TT_ERR_UNSUPPORTED and append(dtype=7) == c.TT_ERR_BAD_DTYPE
    for kw in (dict(page=8), dict(page=24), dict(page=0), dict(hkv=0), dict(pages=-1), dict(pages=1 << 27, page=16), dict(T=-1), dict(T=1 << 30, hkv=2), dict(kc=_at(kc, 8)), dict(vc=_at(vc, 4)),
               dict(vc=kc), dict(vc=_at(kc, 16 * 34 * 2)), dict(k=_at(k, 2)), dict(k=_at(k, 1), dtype=1), dict(ks=(ctypes.c_int64 * 2)(-128, 64)),
               dict(k=kc), dict(v=_at(kc, 3200)), dict(k=_at(vc, -4 * (3 * 128 + 127))), dict(slots=_at(vc, 3200)), dict(pages=2 ** 26, page=16, hkv=256)):
        assert append(**kw) == c.TT_ERR_BAD_SHAPE, kw
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(ks=None), dict(vs=None)):
        assert append(**kw) == c.TT_ERR_NULL, kw

    def read(kc=kc, vc=vc, table=table, cu=cu, B=2, hkv=2, D=64, pages=3, page=16, max_pages=4, total=40, k=ok, v=ov):
        return lib.tt_cache_read_q4(kc, vc, table, cu, B, hkv, D, pages, page, max_pages, total, k, v, None)

    assert read(D=32) == c.TT_ERR_UNSUPPORTED
    for kw in (dict(B=0), dict(max_pages=0), dict(total=-1), dict(total=1 << 30), dict(page=12), dict(hkv=0), dict(k=_at(ok, 2)), dict(v=ok), dict(k=kc), dict(v=_at(vc, 3200)), dict(kc=_at(kc, 1))):
        assert read(**kw) == c.TT_ERR_BAD_SHAPE, kw
    for kw in (dict(table=None), dict(cu=None), dict(k=None), dict(v=None), dict(kc=None)):
        assert read(**kw) == c.TT_ERR_NULL, kw
    if not torch.cuda.is_available():
        assert append() == c.TT_ERR_BAD_DEVICE and read() == c.TT_ERR_BAD_DEVICE
    del raw


def test_q4_format():
    """Every code's scale, the smallest scale that reaches a value, and errors of half a step."""
    import numpy as np
    import q4_oracle as q4
    s = q4.scales(np.arange(q4.TOP + 1))
    assert s[0] == 0 and s[1] == 2.0 ** -20 and s[8] == 2.0 ** -17 and s[q4.TOP] == 896.0 and (np.diff(s) > 0).all() and np.isnan(q4.scales(q4.NAN))
    x = np.random.default_rng(0).standard_normal((50, 2, 64)) * np.logspace(-4, 3, 50)[:, None, None]
    nib, codes = q4.encode(x)
    step = np.repeat(q4.scales(codes), 32, -1)
    assert (np.abs(q4.decode(nib, codes) - x) <= step / 2 * (1 + 1e-12)).all()
    top = np.abs(x.reshape(50, 2, 2, 32)).max(-1)
    assert (7.5 * q4.scales(codes) >= top).all() and (7.5 * q4.scales(codes - 1) < top).all()


def test_q4_decode_refuses_what_does_not_fit(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, p = _buffers(10, 1 << 16)
    q, kc, vc, table, lens, out, ws = p[:7]

    def call(q=q, kc=kc, vc=vc, table=table, pages=9, page=16, max_pages=4, out=out, lse=None, ws=ws, ws_bytes=1 << 16, **kw):
        a = dict(B=2, H=4, S=1, L=50, D=64, dtype=c.TT_BF16, Hkv=2)
        a.update(kw)
        d = c.make_desc(a["B"], a["H"], a["S"], a["L"], a["D"], a["dtype"], False, a.get("scale"), Hkv=a["Hkv"])
        return lib.tt_attn_decode_q4(ctypes.byref(d), q, kc, vc, table, lens, pages, page, max_pages, out, lse, ws, ws_bytes, None)

    for kw in (dict(S=2), dict(L=0), dict(L=65), dict(L=(1 << 30) + 1, max_pages=1 << 27), dict(H=3), dict(B=0), dict(page=8, max_pages=8), dict(page=24), dict(max_pages=3), dict(pages=-1),
               dict(q=_at(q, 2)), dict(out=_at(out, 8)), dict(kc=_at(kc, 8)), dict(table=None, page=48), dict(table=None, page=64, pages=1), dict(scale=math.inf),
               dict(out=q), dict(out=_at(q, 16)), dict(out=_at(kc, 256)), dict(out=vc), dict(lse=out), dict(lse=_at(q, 64)), dict(lse=lens),
               dict(lse=table), dict(pages=2 ** 26, Hkv=128, H=128), dict(B=1 << 20, H=1 << 12)):
        assert call(**kw) == c.TT_ERR_BAD_SHAPE, kw
    for kw in (dict(D=96), dict(dtype=c.TT_F32)):
        assert call(**kw) == c.TT_ERR_BAD_DTYPE, kw
    for kw in (dict(q=None), dict(out=None), dict(kc=None), dict(vc=None)):
        assert call(**kw) == c.TT_ERR_NULL, kw
    assert lib.tt_attn_decode_q4(None, q, kc, vc, table, lens, 9, 16, 4, out, None, ws, 1 << 16, None) == c.TT_ERR_NULL
    long = dict(L=5000, max_pages=313, pages=700)
    d = c.make_desc(2, 4, 1, 5000, 64, c.TT_BF16, False, None, Hkv=2)
    need = lib.tt_attn_decode_q4_workspace_bytes(ctypes.byref(d))
    assert need > 0
    raw2, (big, k_far, v_far) = _buffers(4, 1 << 20)
    assert need < 1 << 20
    for kw in (dict(out=big), dict(out=_at(big, need - 256)), dict(lse=_at(big, 256)), dict(q=_at(big, 512)), dict(table=_at(big, 512))):
        assert call(**long, kc=k_far, vc=v_far, ws=big, ws_bytes=need, **kw) == c.TT_ERR_BAD_SHAPE and "workspace" in c.last_error(), kw
    for L, some in ((1, False), (128, False), (129, True)):
        assert (lib.tt_attn_decode_q4_workspace_bytes(ctypes.byref(c.make_desc(2, 4, 1, L, 64, c.TT_BF16, False, None, Hkv=2))) > 0) == some
    assert call(**long, ws=None) == c.TT_ERR_WORKSPACE and call(**long, ws_bytes=need - 1) == c.TT_ERR_WORKSPACE and call(**long, ws=_at(ws, 64), ws_bytes=need) == c.TT_ERR_WORKSPACE
    if not torch.cuda.is_available():
        assert call() == c.TT_ERR_BAD_DEVICE
    del raw
