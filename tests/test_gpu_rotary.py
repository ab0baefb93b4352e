"""Rotary positions against the formula in 64 bits.

Bound per value, for x1, x2 of its pair and angle t: the angle is off by t 2^-52 (two roundings in 64 bits) and pi 2^-25 (the
reduced turn in 32 bits), sine and cosine by at most 2^-23 each (two units in the last place), their product with scale by
2^-24, the two products and their sum by 2^-24 each; that is under (4e-7 + t 2^-52) scale (|x1| + |x2|), and the output's
rounding is half a step, eps / 2 relative to the value."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def oracle(x, pos, freq, axes, interleaved, scale, back):
    """x [..., D] in 64 bits; pos [A, ...] broadcastable to x's rows -> (result, bound without the output's rounding)."""
    half = len(freq)
    y, bound = x.astype(np.float64) * 1.0, np.zeros(x.shape)
    for i in range(half):
        t = pos[axes[i] if axes is not None else 0].astype(np.float64) * freq[i]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = np.cos(t) * scale, np.sin(t) * scale * (-1 if back else 1)
        x1, x2 = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
        y[..., a], y[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
        bound[..., a] = bound[..., b] = (4e-7 + np.abs(t) * 2.0 ** -52) * abs(scale) * (np.abs(x1) + np.abs(x2))
    return y, bound


def check(got, x, pos, freq, axes, interleaved=False, scale=1.0, back=False):
    want, bound = oracle(x.double().cpu().numpy(), pos, freq.cpu().numpy(), axes.tolist() if axes is not None else None, interleaved, scale, back)
    eps = torch.finfo(got.dtype).eps
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= (bound + eps / 2 * np.abs(want)) * (1 + 1e-6)).all(), float((off - bound - eps / 2 * np.abs(want)).max())


def positions(rng, shape, far):
    p = torch.from_numpy(rng.integers(0, far, shape).astype(np.int32)).cuda()
    return p


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,Hkv,D,R,A", [(1, 1, 1, 64, 64, 1), (1, 32, 8, 128, 128, 1), (7, 4, 2, 128, 64, 3), (33, 5, 1, 80, 80, 2), (130, 3, 3, 96, 24, 4), (9, 2, 2, 256, 256, 1),
                                            (5, 2, 1, 256, 2, 1), (11, 3, 1, 2, 2, 1), (17, 2, 2, 50, 34, 2), (700, 8, 8, 64, 64, 3), (3, 300, 1, 16, 16, 1)])
def test_packed(tt, T, H, Hkv, D, R, A, dtype, interleaved):
    rng = np.random.default_rng(T + D)
    q, k = (torch.randn(T, h, D, device="cuda").to(dtype) for h in (H, Hkv))
    sections = [R // 2 // A + (a < R // 2 % A) for a in range(A)]
    freq, axes = tt.rotary_frequencies(R, sections=sections, cyclic=interleaved)
    pos = positions(rng, (A, T), 100000)
    p = pos.cpu().numpy()[:, :, None]
    for back, call in ((False, tt.rotary_forward), (True, tt.rotary_backward)):
        a, b = call(q, k, pos, freq, axes=axes, interleaved=interleaved)
        check(a, q, p, freq, axes, interleaved, back=back)
        check(b, k, p, freq, axes, interleaved, back=back)
        only, none = call(q, None, pos if A > 1 else pos[0], freq, axes=axes, interleaved=interleaved, scale=0.5)
        assert none is None
        check(only, q, p, freq, axes, interleaved, 0.5, back)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,S,D,R", [(1, 2, 1, 1, 64, 64), (3, 4, 2, 37, 128, 128), (2, 3, 3, 129, 48, 16)])
def test_dense(tt, B, H, Hkv, S, D, R, dtype):
    rng = np.random.default_rng(S)
    q, k = (torch.randn(B, h, S, D, device="cuda").to(dtype) for h in (H, Hkv))
    freq, axes = tt.rotary_frequencies(R, sections=(R // 4, R // 2 - R // 4), own_ladder=True)
    each, shared = positions(rng, (2, B, S), 3000), positions(rng, (2, S), 3000)
    a, b = tt.rotary_forward(q, k, each, freq, axes)
    check(a, q, each.cpu().numpy()[:, :, None], freq, axes)
    check(b, k, each.cpu().numpy()[:, :, None], freq, axes)
    a, b = tt.rotary_backward(q, k, shared, freq, axes)
    check(a, q, shared.cpu().numpy()[:, None, None], freq, axes, back=True)
    one, _ = tt.rotary_forward(q, None, shared[0], freq)
    check(one, q, shared.cpu().numpy()[:1, None, None], freq, None)


def test_strides_alignment_and_repeats(tt):
    rng = np.random.default_rng(3)
    S, H, Hkv, D = 53, 6, 2, 64
    freq, axes = tt.rotary_frequencies(D, sections=(16, 8, 8))
    pos = positions(rng, (3, S), 5000)
    p = pos.cpu().numpy()[:, :, None]
    rows = torch.randn(S, H + 2 * Hkv, D, device="cuda").bfloat16()       # slices of a projection
    a, b = tt.rotary_forward(rows[:, :H], rows[:, H:H + Hkv], pos, freq, axes)
    check(a, rows[:, :H], p, freq, axes)
    check(b, rows[:, H:H + Hkv], p, freq, axes)
    odd = torch.randn(S, H, D + 1, device="cuda").bfloat16()                # rows off 16 bytes
    check(tt.rotary_forward(odd[..., 1:], None, pos, freq, axes)[0], odd[..., 1:], p, freq, axes)
    off = torch.randn(S * H * D + 1, device="cuda").bfloat16()[1:].view(S, H, D)
    check(tt.rotary_forward(off, None, pos, freq, axes)[0], off, p, freq, axes)
    x = torch.randn(1, H, S, D, device="cuda")
    many = x.expand(4, H, S, D)                                             # one batch entry shown four times
    where = positions(rng, (1, 4, S), 5000)
    f1, _ = tt.rotary_frequencies(D)
    check(tt.rotary_forward(many, None, where, f1)[0], many, where.cpu().numpy()[:, :, None], f1, None)
    same = pos[:1].expand(3, S)                                             # text: one position on all axes
    check(tt.rotary_forward(off, None, same, freq, axes)[0], off, same.cpu().numpy()[:, :, None], freq, axes)
    turned = torch.randn(S, H, D, device="cuda").transpose(0, 1).contiguous().transpose(0, 1)   # head-major rows
    check(tt.rotary_forward(turned, None, pos, freq, axes)[0], turned, p, freq, axes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R", [64, 24])
def test_in_place_and_into_slices(tt, dtype, R):
    S, H, Hkv, D = 41, 4, 2, 64
    freq, axes = tt.rotary_frequencies(R)
    pos = torch.arange(S, dtype=torch.int32, device="cuda") * 77
    rows = torch.randn(S, H + 2 * Hkv, D, device="cuda").to(dtype)
    want = tt.rotary_forward(rows[:, :H], rows[:, H:H + Hkv], pos, freq)
    other = torch.full_like(rows, 7.0)
    tt.rotary_forward(rows[:, :H], rows[:, H:H + Hkv], pos, freq, out_q=other[:, :H], out_k=other[:, H:H + Hkv])
    assert torch.equal(other[:, :H], want[0]) and torch.equal(other[:, H:H + Hkv], want[1]) and (other[:, H + Hkv:] == 7.0).all()
    v = rows[:, H + Hkv:].clone()
    got = tt.rotary_forward(rows[:, :H], rows[:, H:H + Hkv], pos, freq, out_q=rows[:, :H], out_k=rows[:, H:H + Hkv])
    assert torch.equal(rows[:, :H], want[0]) and torch.equal(rows[:, H:H + Hkv], want[1]) and torch.equal(rows[:, H + Hkv:], v)
    assert got[0].data_ptr() == rows.data_ptr()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,R,shift,gap", [(80, 20, 0, 0), (80, 40, 0, 0), (64, 12, 0, 0), (128, 128, 4, 0), (128, 64, 2, 4), (96, 96, 0, 2), (128, 128, 0, 4), (82, 82, 0, 0), (64, 64, 1, 0)])
def test_every_width_of_access(tt, D, R, shift, gap, dtype, interleaved):
    """Rows that begin, end or halve at 2, 4 or 8 bytes; the output's rows too, with what lies between them left as it was."""
    T, H = 29, 3
    whole = torch.randn(T * H * (D + gap) + shift, device="cuda").to(dtype)
    x = whole[shift:].view(T, H, D + gap)[..., :D]
    freq, _ = tt.rotary_frequencies(R)
    pos = positions(np.random.default_rng(D + R), (1, T), 3000)
    p = pos.cpu().numpy()[:, :, None]
    check(tt.rotary_forward(x, None, pos, freq, interleaved=interleaved)[0], x, p, freq, None, interleaved)
    into = torch.full_like(whole, 7)
    y = into[shift:].view(T, H, D + gap)
    got, _ = tt.rotary_backward(x, None, pos, freq, interleaved=interleaved, out_q=y[..., :D])
    check(got, x, p, freq, None, interleaved, back=True)
    assert got.data_ptr() == y.data_ptr() and (y[..., D:] == 7).all() and (into[:shift] == 7).all()


def test_far_and_negative_positions(tt):
    pos = torch.tensor([0, 1, -1, 2 ** 20 + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    x = torch.randn(6, 2, 128, device="cuda")
    freq, _ = tt.rotary_frequencies(128)
    got, _ = tt.rotary_forward(x, None, pos, freq)
    check(got, x, pos.cpu().numpy()[None, :, None], freq, None)
    assert torch.equal(got[0], x[0])
    freq[3] = 0.0
    assert torch.equal(tt.rotary_forward(x, None, pos, freq)[0][:, :, 3], x[:, :, 3])


def test_axes_outside_are_taken_as_the_nearest(tt):
    x = torch.randn(5, 1, 8, device="cuda")
    freq, _ = tt.rotary_frequencies(8)
    pos = torch.randint(0, 99, (2, 5), dtype=torch.int32, device="cuda")
    far = torch.tensor([-5, 0, 1, 2 ** 30], dtype=torch.int32, device="cuda")
    near = torch.tensor([0, 0, 1, 1], dtype=torch.int32, device="cuda")
    assert torch.equal(tt.rotary_forward(x, None, pos, freq, far)[0], tt.rotary_forward(x, None, pos, freq, near)[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(tt, interleaved):
    """The map is linear: a central difference is exact but for roundings, 2^-24 of values of size 4 over a step of 1, twice."""
    T, H, D = 3, 2, 12
    x, g = torch.randn(T, H, D, device="cuda"), torch.randn(T, H, D, device="cuda")
    freq, axes = tt.rotary_frequencies(8, sections=(1, 3))
    pos = torch.randint(0, 1000, (2, T), dtype=torch.int32, device="cuda")
    call = lambda z: tt.rotary_forward(z, None, pos, freq, axes, interleaved, 1.5)[0].double()
    dx, _ = tt.rotary_backward(g, None, pos, freq, axes, interleaved, 1.5)
    for i in range(x.numel()):
        step = torch.zeros_like(x).view(-1)
        step[i] = 1.0
        step = step.view_as(x)
        slope = float(((call(x + step) - call(x - step)) / 2 * g.double()).sum())
        assert abs(slope - float(dx.view(-1)[i])) < 3e-5


def test_streams_and_graphs(tt):
    T, H, D = 200, 4, 128
    freq, axes = tt.rotary_frequencies(D, sections=(20, 22, 22))
    x, pos = torch.randn(T, H, D, device="cuda").bfloat16(), torch.randint(0, 9999, (3, T), dtype=torch.int32, device="cuda")
    want, _ = tt.rotary_forward(x, None, pos, freq, axes)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs.append(tt.rotary_forward(x, None, pos, freq, axes)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = tt.rotary_forward(x, None, pos, freq, axes)
        back, _ = tt.rotary_backward(y, None, pos, freq, axes)
    x.copy_(torch.randn(T, H, D, device="cuda"))
    pos.random_(0, 100)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, tt.rotary_forward(x, None, pos, freq, axes)[0]) and torch.equal(back, tt.rotary_backward(y, None, pos, freq, axes)[0])


def test_empty_and_refusals(tt):
    freq, axes = tt.rotary_frequencies(64, sections=(16, 16))
    x = torch.randn(4, 2, 64, device="cuda")
    pos = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    e, _ = tt.rotary_forward(x[:0], None, pos[:, :0], freq, axes)
    assert e.shape == (0, 2, 64)
    for kw in (dict(q=x.half()), dict(q=x.cpu()), dict(q=x[0]), dict(q=x.transpose(1, 2)), dict(k=x.bfloat16()), dict(k=x[:3]), dict(k=x[..., :32]), dict(positions=pos.long()),
               dict(positions=pos[:, :3]), dict(positions=pos[None]), dict(positions=pos.t().contiguous().t()), dict(inv_freq=freq.float()), dict(inv_freq=freq[None]),
               dict(axes=axes[:5]), dict(axes=axes.long()), dict(out_q=x[:, :1]), dict(out_q=torch.empty(4, 2, 64, device="cuda").expand(4, 2, 64)[:1].expand(4, 2, 64)),
               dict(out_k=x), dict(inv_freq=torch.ones(33, dtype=torch.float64, device="cuda"), axes=None), dict(scale=float("nan"))):
        a = dict(q=x, k=None, positions=pos, inv_freq=freq, axes=axes)
        a.update(kw)
        with pytest.raises(ValueError):
            tt.rotary_forward(**a)
    with pytest.raises(TypeError):
        tt.rotary_forward(x, None, pos, freq, axes, scale=[1])


def test_neighbouring_memory_stays(tt):
    from test_gpu_canary import Guarded
    for dtype in (torch.bfloat16, torch.float32):
        for T, H, D, R in ((1, 1, 64, 64), (13, 3, 80, 40), (129, 2, 128, 128)):
            q, out = Guarded((T, H, D), dtype, torch.randn(T, H, D)), Guarded((T, H, D), dtype)
            freq, _ = tt.rotary_frequencies(R)
            tt.rotary_forward(q.t, None, torch.arange(T, dtype=torch.int32, device="cuda"), freq, out_q=out.t)
            torch.cuda.synchronize()
            assert q.intact() and out.intact()


def test_frequencies_beyond_a_turn_and_not_finite(tt):
    """Several turns a position, half a turn exactly, both signs; a frequency that is no number makes its pair so and no other."""
    freq = torch.tensor([100.0, -7.0, np.pi, -np.pi, 1e-30, 2e5, float("nan"), float("inf")], dtype=torch.float64, device="cuda")
    pos = torch.tensor([0, 1, 3, -5, 123456, -99999], dtype=torch.int32, device="cuda")
    x = torch.randn(6, 2, 20, device="cuda")
    got, _ = tt.rotary_forward(x, None, pos, freq, interleaved=True)
    assert got[..., 12:16].isnan().all() and torch.equal(got[..., 16:], x[..., 16:])
    check(torch.cat([got[..., :12], got[..., 16:]], -1), torch.cat([x[..., :12], x[..., 16:]], -1), pos.cpu().numpy()[None, :, None], freq[:6], None, True)
