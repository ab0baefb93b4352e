"""Argument checks of the normed heads and of appending with rotation (status codes, no GPU needed), and the gradient's formula against differences."""
import ctypes

import numpy as np
import pytest

import norm_rotary_oracle as nr


def _desc(tt, **kw):
    d = tt.capi.RotaryDesc(B=2, S=4, H=4, Hkv=2, D=64, R=32, n_axes=1, dtype=tt.capi.TT_F32, interleaved=0, scale=1.0)
    d.q_stride = d.q_out_stride = (4 * 4 * 64, 4 * 64, 64)
    d.k_stride = d.k_out_stride = (2 * 4 * 64, 4 * 64, 64)
    d.pos_stride = (8, 4)
    for name, value in kw.items():
        setattr(d, name, value)
    return d


BASE = ctypes.addressof(ctypes.create_string_buffer(1 << 20, 1 << 20)) // 256 * 256 + 256


def _at(i):
    return ctypes.c_void_p(BASE + (i << 14))


def test_forward_refuses_what_does_not_fit(tt):
    c, lib = tt.capi, tt.capi.lib

    def call(d, q=_at(0), k=_at(1), wq=_at(2), wk=_at(3), wt=0, eps=1e-6, pos=_at(4), freq=_at(5), q_out=_at(6), k_out=_at(7)):
        return lib.tt_norm_rotary(ctypes.byref(d) if d is not None else None, q, k, wq, wk, wt, eps, pos, freq, None, q_out, k_out, None)

    assert call(_desc(tt)) == c.TT_ERR_BAD_DEVICE   # all that is missing is a GPU
    assert call(None) == c.TT_ERR_NULL
    for name in ("q", "wq", "wk", "pos", "freq", "q_out", "k_out"):
        assert call(_desc(tt), **{name: None}) == c.TT_ERR_NULL, name
    assert call(_desc(tt), k=None, k_out=None, wk=None) == c.TT_ERR_BAD_DEVICE
    for bad in (dict(D=1), dict(D=257), dict(R=0), dict(R=31), dict(R=66), dict(H=0), dict(Hkv=0), dict(n_axes=0), dict(B=-1), dict(S=-1), dict(scale=float("inf"))):
        assert call(_desc(tt, **bad)) == c.TT_ERR_BAD_SHAPE, bad
    for eps in (0.0, -1e-6, float("nan"), float("inf")):
        assert call(_desc(tt), eps=eps) == c.TT_ERR_BAD_SHAPE
    assert call(_desc(tt), wt=7) == c.TT_ERR_BAD_DTYPE and call(_desc(tt, dtype=5)) == c.TT_ERR_BAD_DTYPE
    assert call(_desc(tt), wq=ctypes.c_void_p(BASE + (2 << 14) + 2)) == c.TT_ERR_BAD_SHAPE
    assert call(_desc(tt), wq=_at(6)) == c.TT_ERR_BAD_SHAPE and call(_desc(tt), wk=_at(6)) == c.TT_ERR_BAD_SHAPE
    assert call(_desc(tt), q_out=_at(1)) == c.TT_ERR_BAD_SHAPE and call(_desc(tt), pos=_at(6)) == c.TT_ERR_BAD_SHAPE
    assert call(_desc(tt), q_out=_at(0), k_out=_at(1)) == c.TT_ERR_BAD_DEVICE   # in place
    assert call(_desc(tt, S=0), q=None, pos=None) == c.TT_OK


def test_backward_refuses_what_does_not_fit(tt):
    c, lib = tt.capi, tt.capi.lib
    st = (ctypes.c_int64 * 3)(4 * 4 * 64, 4 * 64, 64)
    names = dict(dq=0, dk=1, q=2, k=3, wq=4, wk=5, pos=6, freq=7, dq_out=8, dk_out=9, dwq=10, dwk=11, ws=12)

    def call(d, eps=1e-6, wt=0, st=st, n=1 << 14, **kw):
        p = {**{name: _at(i) for name, i in names.items()}, **kw}
        return lib.tt_norm_rotary_bwd(ctypes.byref(d), p["dq"], p["dk"], p["q"], p["k"], st, (ctypes.c_int64 * 3)(2 * 4 * 64, 4 * 64, 64), p["wq"], p["wk"], wt, eps, p["pos"],
                                      p["freq"], None, p["dq_out"], p["dk_out"], p["dwq"], p["dwk"], p["ws"], n, None)

    assert call(_desc(tt)) == c.TT_ERR_BAD_DEVICE
    for name in names:
        if name != "ws":   # (asked for once the device is known)
            assert call(_desc(tt), **{name: None}) == c.TT_ERR_NULL, name
    assert call(_desc(tt), dk=None, k=None, wk=None, dk_out=None, dwk=None) == c.TT_ERR_BAD_DEVICE
    assert call(_desc(tt), eps=0.0) == c.TT_ERR_BAD_SHAPE and call(_desc(tt), wt=3) == c.TT_ERR_BAD_DTYPE
    assert call(_desc(tt), st=(ctypes.c_int64 * 3)(-1, 256, 64)) == c.TT_ERR_BAD_SHAPE
    assert call(_desc(tt), dq_out=_at(0), dk_out=_at(1)) == c.TT_ERR_BAD_DEVICE   # onto the upstream gradients
    for a, b in (("dq_out", "q"), ("dk_out", "k"), ("dq_out", "k"), ("dk_out", "q"), ("dq_out", "dk"), ("dq_out", "dk_out"), ("dwq", "q"), ("dwk", "dq"), ("dwq", "dwk"),
                 ("ws", "dq_out"), ("ws", "dwk"), ("dwq", "wq"), ("dwk", "pos"), ("dwq", "freq"), ("dq_out", "wk"), ("ws", "k"), ("dwk", "dk_out")):
        assert call(_desc(tt), **{a: _at(names[b])}) == c.TT_ERR_BAD_SHAPE, (a, b)
    assert call(_desc(tt), dwq=ctypes.c_void_p(BASE + (10 << 14) + 1)) == c.TT_ERR_BAD_SHAPE


def test_append_refuses_what_does_not_fit(tt):
    c, lib = tt.capi, tt.capi.lib
    names = dict(q=0, k=1, v=2, slots=3, pos=4, freq=5, wq=6, wk=7, q_out=8, k_out=9, kp=10, vp=12)

    def desc(**kw):
        d = _desc(tt, B=1, dtype=c.TT_BF16, pos_stride=(4, 4), q_stride=(0, 64, 256), q_out_stride=(0, 64, 256), k_stride=(0, 64, 128), k_out_stride=(0, 64, 128))
        for name, value in kw.items():
            setattr(d, name, value)
        return d

    def call(d, wt=0, eps=1e-6, vs=(128, 64), pages=5, page=16, **kw):
        p = {**{name: _at(i) for name, i in names.items()}, **kw}
        return lib.tt_cache_append_rotary(ctypes.byref(d), p["q"], p["k"], p["v"], (ctypes.c_int64 * 2)(*vs), p["slots"], p["pos"], p["freq"], None, p["wq"], p["wk"], wt,
                                          eps, p["q_out"], p["k_out"], p["kp"], p["vp"], pages, page, None)

    assert call(desc()) == c.TT_ERR_BAD_DEVICE and call(desc(), wq=None, wk=None) == c.TT_ERR_BAD_DEVICE
    assert call(desc(), q=None, q_out=None) == c.TT_ERR_BAD_DEVICE and call(desc(), k_out=None) == c.TT_ERR_BAD_DEVICE
    for name in ("q", "k", "v", "slots", "pos", "freq", "wq", "wk", "q_out", "kp", "vp"):
        assert call(desc(), **{name: None}) == c.TT_ERR_NULL, name
    for bad in (dict(B=2), dict(Hkv=0), dict(R=66), dict(n_axes=0)):
        assert call(desc(**bad)) == c.TT_ERR_BAD_SHAPE, bad
    assert call(desc(D=32, R=32)) == c.TT_ERR_UNSUPPORTED
    for bad in (dict(page=0), dict(pages=-1), dict(pages=1 << 20, page=1 << 12), dict(vs=(-1, 64)), dict(eps=0.0), dict(wk=ctypes.c_void_p(BASE + (7 << 14) + 2))):
        assert call(desc(), **bad) == c.TT_ERR_BAD_SHAPE, bad
    assert call(desc(), q_out=_at(0), k_out=_at(1)) == c.TT_ERR_BAD_DEVICE
    assert call(desc(dtype=c.TT_F32), q_out=_at(0)) == c.TT_ERR_BAD_SHAPE   # floats are not turned in place
    for a, b in (("q_out", "k"), ("k_out", "v"), ("q_out", "k_out"), ("kp", "k"), ("vp", "q"), ("kp", "vp"), ("vp", "slots"), ("kp", "wq"), ("q_out", "kp"), ("k_out", "slots"),
                 ("k_out", "pos"), ("q_out", "wk"), ("vp", "freq")):
        assert call(desc(), **{a: _at(names[b])}) == c.TT_ERR_BAD_SHAPE, (a, b)


@pytest.mark.parametrize("interleaved", [False, True])
def test_formula_against_differences(interleaved):
    rng = np.random.default_rng(8)
    x, w, c, t = rng.standard_normal((3, 2, 12)), rng.standard_normal(12), rng.standard_normal((3, 2, 12)), rng.uniform(0, 6, (3, 1, 4))
    dx, _, dw, _ = nr.backward(c, x, w, t, interleaved, 1.5, 0.1)
    loss = lambda x, w: (nr.forward(x, w, t, interleaved, 1.5, 0.1)[0] * c).sum()
    h = 1e-6
    for i in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[i] = h
        assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * h) - dx[i]) < 1e-7
    for i in range(12):
        e = np.zeros(12)
        e[i] = h
        assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - dw[i]) < 1e-7
