"""Outputs on the arrays that say where rows are and how far they turn: refused, since some CTAs would look there after others have written."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def _buffers(n, size=1 << 14):
    raw = (ctypes.c_char * ((n + 1) * size))()
    base = ctypes.addressof(raw)
    base += -base % 256
    return raw, [ctypes.c_void_p(base + i * size) for i in range(n)]


def _at(p, offset):
    return ctypes.c_void_p(p.value + offset)


def test_reading_the_cache_onto_its_tables(tt):
    lib, c = tt.capi.lib, tt.capi
    raw, (kc, vc, table, cu, k, v) = _buffers(6)
    B, hkv, D, pages, page, width, total = 2, 1, 64, 3, 16, 4, 40

    def read(table=table, cu=cu, k=k, v=v):
        return lib.tt_cache_read_q4(kc, vc, table, cu, B, hkv, D, pages, page, width, total, k, v, None)

    size = total * hkv * D * 2
    for kw in (dict(k=table), dict(v=table), dict(k=cu), dict(v=cu), dict(table=_at(k, size - 4)), dict(table=_at(v, -(B * width * 4 - 4))), dict(cu=_at(v, size - 4)),
               dict(cu=_at(k, -4 * B))):
        assert read(**kw) == c.TT_ERR_BAD_SHAPE and "overlaps" in c.last_error(), kw
    if not torch.cuda.is_available():
        for kw in (dict(), dict(table=_at(k, size)), dict(table=_at(v, -B * width * 4)), dict(cu=_at(v, size)), dict(cu=_at(k, -4 * (B + 1)))):
            assert read(**kw) == c.TT_ERR_BAD_DEVICE, kw
    del raw


@pytest.mark.parametrize("with_k", [True, False])
def test_rotary_onto_its_positions_and_frequencies(tt, with_k):
    lib, c = tt.capi.lib, tt.capi
    raw, (q, k, q_out, k_out, pos, freq, axes) = _buffers(7)
    B, S, H, hkv, D, R, A = 2, 4, 3, 2, 16, 8, 2
    d = c.RotaryDesc(B=B, S=S, H=H, Hkv=hkv, D=D, R=R, n_axes=A, dtype=c.TT_F32, interleaved=0, scale=1.0)
    d.q_stride[:] = d.q_out_stride[:] = (H * S * D, S * D, D)
    d.k_stride[:] = d.k_out_stride[:] = (hkv * S * D, S * D, D)
    d.pos_stride[:] = (B * S, S)

    def turn(q_out=q_out, k_out=k_out, pos=pos, freq=freq, axes=axes):
        return lib.tt_rotary(ctypes.byref(d), q, k if with_k else None, pos, freq, axes, 0, q_out, k_out if with_k else None, None)

    nq, nk, n_pos = B * H * S * D * 4, B * hkv * S * D * 4, A * B * S * 4
    bad = [dict(q_out=pos), dict(q_out=freq), dict(q_out=axes), dict(pos=_at(q_out, nq - 4)), dict(pos=_at(q_out, 4 - n_pos)), dict(freq=_at(q_out, nq - 8)),
           dict(freq=_at(q_out, 8 - 4 * R)), dict(axes=_at(q_out, nq - 4)), dict(axes=_at(q_out, 4 - 2 * R))]
    if with_k:
        bad += [dict(k_out=pos), dict(k_out=freq), dict(k_out=axes), dict(pos=_at(k_out, nk - 4)), dict(freq=_at(k_out, 8 - 4 * R)), dict(axes=_at(k_out, nk - 4))]
    for kw in bad:
        assert turn(**kw) == c.TT_ERR_BAD_SHAPE and "overlaps" in c.last_error(), kw
    if not torch.cuda.is_available():
        for kw in (dict(), dict(axes=None), dict(pos=_at(q_out, nq)), dict(pos=_at(q_out, -n_pos)), dict(freq=_at(q_out, nq)), dict(axes=_at(q_out, -2 * R))):
            assert turn(**kw) == c.TT_ERR_BAD_DEVICE, kw
        # positions that repeat along axes and batch
        d.pos_stride[:] = (0, 0)
        assert turn(pos=_at(q_out, -4 * S)) == c.TT_ERR_BAD_DEVICE and turn(pos=_at(q_out, -4 * S + 4)) == c.TT_ERR_BAD_SHAPE
    del raw
