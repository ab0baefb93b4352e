"""Argument checks of the 8-bit cache's calls (status codes, no GPU needed) and its format."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")


def _buffers(n=8, size=4096):
    raw = (ctypes.c_char * (n * size))()
    base = ctypes.addressof(raw)
    base += -base % 256
    return raw, [ctypes.c_void_p(base + i * size) for i in range(n - 1)]


def _at(p, offset):
    return ctypes.c_void_p(p.value + offset)


def test_q8_cache_refuses_what_does_not_fit(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, p = _buffers(10, 1 << 16)
    k, v, slots, kc, vc, table, cu, ok, ov = p[:9]
    st = (ctypes.c_int64 * 2)(128, 64)
    assert [lib.tt_cache_q8_page_bytes(*a) for a in ((16, 64), (48, 128), (8, 64), (24, 64), (16, 96), (0, 64), (-16, 128))] == [16 * 64 + 32, 48 * 128 + 32, 0, 0, 0, 0, 0]

    def append(k=k, v=v, slots=slots, T=4, hkv=2, D=64, dtype=0, ks=st, vs=st, kc=kc, vc=vc, pages=3, page=16):
        return lib.tt_cache_append_q8(k, v, slots, T, hkv, D, dtype, ks, vs, kc, vc, pages, page, None)

    assert append(D=96) == c.TT_ERR_UNSUPPORTED and append(dtype=7) == c.TT_ERR_BAD_DTYPE
    for kw in (dict(page=8), dict(page=24), dict(page=0), dict(hkv=0), dict(pages=-1), dict(pages=1 << 27, page=16), dict(T=-1), dict(T=1 << 30, hkv=2), dict(kc=_at(kc, 8)), dict(vc=_at(vc, 4)),
               dict(vc=kc), dict(vc=_at(kc, 1056 * 2)), dict(k=_at(k, 2)), dict(k=_at(k, 1), dtype=1), dict(ks=(ctypes.c_int64 * 2)(-128, 64)),
               dict(k=kc), dict(v=_at(kc, 6200)), dict(k=_at(vc, -4 * (3 * 128 + 127))), dict(slots=_at(vc, 6200)), dict(pages=2 ** 26, page=16, hkv=256)):
        assert append(**kw) == c.TT_ERR_BAD_SHAPE, kw
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(ks=None), dict(vs=None)):
        assert append(**kw) == c.TT_ERR_NULL, kw

    def read(kc=kc, vc=vc, table=table, cu=cu, B=2, hkv=2, D=64, pages=3, page=16, max_pages=4, total=40, k=ok, v=ov):
        return lib.tt_cache_read_q8(kc, vc, table, cu, B, hkv, D, pages, page, max_pages, total, k, v, None)

    assert read(D=32) == c.TT_ERR_UNSUPPORTED
    for kw in (dict(B=0), dict(max_pages=0), dict(total=-1), dict(total=1 << 30), dict(page=12), dict(hkv=0), dict(k=_at(ok, 2)), dict(v=ok), dict(k=kc), dict(v=_at(vc, 6200)), dict(kc=_at(kc, 1))):
        assert read(**kw) == c.TT_ERR_BAD_SHAPE, kw
    for kw in (dict(table=None), dict(cu=None), dict(k=None), dict(v=None), dict(kc=None)):
        assert read(**kw) == c.TT_ERR_NULL, kw
    if not torch.cuda.is_available():
        assert append() == c.TT_ERR_BAD_DEVICE and read() == c.TT_ERR_BAD_DEVICE
    del raw


def test_q8_decode_refuses_what_does_not_fit(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, p = _buffers(10, 1 << 16)
    q, kc, vc, table, lens, out, ws = p[:7]

    def call(q=q, kc=kc, vc=vc, table=table, pages=9, page=16, max_pages=4, out=out, lse=None, ws=ws, ws_bytes=1 << 16, **kw):
        a = dict(B=2, H=4, S=1, L=50, D=64, dtype=c.TT_BF16, Hkv=2)
        a.update(kw)
        d = c.make_desc(a["B"], a["H"], a["S"], a["L"], a["D"], a["dtype"], False, a.get("scale"), Hkv=a["Hkv"])
        return lib.tt_attn_decode_q8(ctypes.byref(d), q, kc, vc, table, lens, pages, page, max_pages, out, lse, ws, ws_bytes, None)

    for kw in (dict(S=2), dict(L=0), dict(L=65), dict(L=(1 << 30) + 1, max_pages=1 << 27), dict(H=3), dict(B=0), dict(page=8, max_pages=8), dict(page=24), dict(max_pages=3), dict(pages=-1),
               dict(q=_at(q, 2)), dict(out=_at(out, 8)), dict(kc=_at(kc, 8)), dict(table=None, page=48), dict(table=None, page=64, pages=1), dict(scale=math.inf),
               dict(out=q), dict(out=_at(q, 16)), dict(out=_at(kc, 256)), dict(out=vc), dict(lse=out), dict(lse=_at(q, 64)), dict(lse=lens),
               dict(lse=table), dict(pages=2 ** 26, Hkv=128, H=128), dict(B=1 << 20, H=1 << 12)):
        assert call(**kw) == c.TT_ERR_BAD_SHAPE, kw
    for kw in (dict(D=96), dict(dtype=c.TT_F32)):
        assert call(**kw) == c.TT_ERR_BAD_DTYPE, kw
    for kw in (dict(q=None), dict(out=None), dict(kc=None), dict(vc=None)):
        assert call(**kw) == c.TT_ERR_NULL, kw
    assert lib.tt_attn_decode_q8(None, q, kc, vc, table, lens, 9, 16, 4, out, None, ws, 1 << 16, None) == c.TT_ERR_NULL
    long = dict(L=5000, max_pages=313, pages=700)
    d = c.make_desc(2, 4, 1, 5000, 64, c.TT_BF16, False, None, Hkv=2)
    need = lib.tt_attn_decode_q8_workspace_bytes(ctypes.byref(d))
    assert need > 0
    raw2, (big, k_far, v_far) = _buffers(4, 1 << 20)
    assert need < 1 << 20
    for kw in (dict(out=big), dict(out=_at(big, need - 256)), dict(lse=_at(big, 256)), dict(q=_at(big, 512)), dict(table=_at(big, 512))):
        assert call(**long, kc=k_far, vc=v_far, ws=big, ws_bytes=need, **kw) == c.TT_ERR_BAD_SHAPE and "workspace" in c.last_error(), kw
    for L, some in ((1, False), (192, False), (193, True)):
        assert (lib.tt_attn_decode_q8_workspace_bytes(ctypes.byref(c.make_desc(2, 4, 1, L, 64, c.TT_BF16, False, None, Hkv=2))) > 0) == some
    assert call(**long, ws=None) == c.TT_ERR_WORKSPACE and call(**long, ws_bytes=need - 1) == c.TT_ERR_WORKSPACE and call(**long, ws=_at(ws, 64), ws_bytes=need) == c.TT_ERR_WORKSPACE
    if not torch.cuda.is_available():
        assert call() == c.TT_ERR_BAD_DEVICE
    del raw


def test_q8_format():
    """All codes in order, the smallest exponent that reaches a value, errors of half a step, and blocks that grow."""
    import numpy as np
    import q8_oracle as q8
    assert q8.POSITIVE[1] == 2.0 ** -9 and q8.POSITIVE[8] == 2.0 ** -6 and q8.POSITIVE[126] == 448 and (np.diff(q8.POSITIVE) > 0).all()
    real = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(real, q8.CODES, equal_nan=True)
    x = np.concatenate([np.random.default_rng(0).standard_normal(2000) * 300, (q8.POSITIVE[1:] + q8.POSITIVE[:-1]) / 2, q8.POSITIVE]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(np.concatenate([x, -x])).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(q8.nearest(np.concatenate([x, -x])), want)
    y = np.random.default_rng(1).standard_normal((40, 16, 2, 64)) * np.logspace(-9, 9, 40)[:, None, None, None]
    for block in y:
        e = q8.exponent(block)
        top = np.abs(block).max((0, 2))
        assert (448 * 2.0 ** e >= top).all() and (448 * 2.0 ** (e - 1) < top).all()
        pool = q8.Pool(1, 2, 16, 64)
        pool.write(np.arange(16), block)
        once = pool.rows([0], 16)
        s = 2.0 ** e[None, :, None]
        assert (np.abs(once - block) <= np.maximum(np.abs(block) * 2.0 ** -4, 2.0 ** -10 * s) * (1 + 1e-12)).all()
        pool = q8.Pool(1, 2, 16, 64)
        for r in range(16):
            pool.write([r], block[r:r + 1])
        assert (np.abs(pool.rows([0], 16) - block) <= np.maximum(np.abs(block) * 2.0 ** -4, 2.0 ** -9 * s) * (1 + 1e-12)).all()
