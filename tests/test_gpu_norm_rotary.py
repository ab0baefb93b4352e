"""Normed heads with rotary positions, forward and backward, against 64 bits; the bounds are those of norm_rotary_oracle."""
import numpy as np
import pytest

import norm_rotary_oracle as nr

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def host(x):
    return x.detach().double().cpu().numpy()


def near(got, want, bound):
    ok, worst = nr.within(host(got), want, bound, torch.finfo(got.dtype).eps)
    assert ok, worst


def angles(pos, freq, axes, dense):
    p = pos.cpu().numpy()
    p = p if p.ndim > 1 else p[None]
    t = nr.angles(p, freq.tolist(), axes.tolist() if axes is not None else None)
    return t if dense and t.ndim == 2 else np.expand_dims(t, 1)   # the same for every head


def weights(D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(D, generator=g)).to(dtype).cuda()


def check(tt, q, k, pos, freq, axes=None, interleaved=False, scale=None, eps=1e-6, wtype=torch.float32, back=True):
    D, dense = q.shape[-1], q.dim() == 4
    wq, wk = weights(D, wtype, 1), weights(D, wtype, 2) if k is not None else None
    t = angles(pos, freq, axes, dense)
    s = 1.0 if scale is None else scale
    how = dict(axes=axes, interleaved=interleaved, eps=eps, scale=scale)
    got = tt.norm_rotary_forward(q, k, wq, wk, pos, freq, **how)
    for y, x, w in zip(got, (q, k), (wq, wk)):
        if x is None:
            assert y is None
            continue
        assert y.dtype == x.dtype and y.shape == x.shape
        near(y, *nr.forward(host(x), host(w), t, interleaved, s, eps))
    if not back:
        return
    dq, dk = torch.randn(q.shape, device="cuda").to(q.dtype), torch.randn(k.shape, device="cuda").to(q.dtype) if k is not None else None
    got = tt.norm_rotary_backward(dq, dk, q, k, wq, wk, pos, freq, **how)
    again = tt.norm_rotary_backward(dq, dk, q, k, wq, wk, pos, freq, **how)
    for i, (dz, x, w) in enumerate(((dq, q, wq), (dk, k, wk))):
        if x is None:
            assert got[i] is None and got[2 + i] is None
            continue
        dx, edx, dw, edw = nr.backward(host(dz), host(x), host(w), t, interleaved, s, eps)
        near(got[i], dx, edx)
        near(got[2 + i], dw, edw)
        assert got[2 + i].dtype == wtype and torch.equal(got[i], again[i]) and torch.equal(got[2 + i], again[2 + i])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,Hkv,D,R,A", [(1, 1, 1, 64, 64, 1), (1, 32, 8, 128, 128, 1), (7, 4, 2, 128, 64, 3), (33, 5, 1, 80, 80, 2), (130, 3, 3, 96, 24, 4), (9, 2, 2, 256, 256, 1),
                                            (5, 2, 1, 256, 2, 1), (11, 3, 1, 2, 2, 1), (17, 2, 2, 50, 34, 2), (300, 8, 8, 64, 64, 3), (3, 300, 1, 16, 16, 1), (6, 1, 70, 65, 12, 1),
                                            (4, 2, 2, 255, 254, 1), (5, 3, 1, 256, 4, 1)])
def test_packed(tt, T, H, Hkv, D, R, A, dtype, interleaved):
    rng = np.random.default_rng(T + D)
    q, k = (torch.randn(T, h, D, device="cuda").to(dtype) for h in (H, Hkv))
    sections = [R // 2 // A + (a < R // 2 % A) for a in range(A)]
    freq, axes = tt.rotary_frequencies(R, sections=sections, cyclic=interleaved)
    pos = torch.from_numpy(rng.integers(0, 100000, (A, T)).astype(np.int32)).cuda()
    check(tt, q, k, pos, freq, axes, interleaved, wtype=dtype)
    check(tt, q, None, pos if A > 1 else pos[0], freq, axes, interleaved, scale=0.5, eps=0.25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,S,D,R", [(1, 2, 1, 1, 64, 64), (3, 4, 2, 37, 128, 128), (2, 3, 3, 129, 48, 16)])
def test_dense(tt, B, H, Hkv, S, D, R, dtype):
    rng = np.random.default_rng(S)
    q, k = (torch.randn(B, h, S, D, device="cuda").to(dtype) for h in (H, Hkv))
    freq, axes = tt.rotary_frequencies(R, sections=(R // 4, R // 2 - R // 4), own_ladder=True)
    for shape in ((2, B, S), (2, S)):
        check(tt, q, k, torch.from_numpy(rng.integers(0, 3000, shape).astype(np.int32)).cuda(), freq, axes)


def test_many_rows(tt):
    """More tiles than CTAs, and a number of tokens that no tile divides."""
    T, H, Hkv, D = 4099, 6, 2, 128
    q, k = (torch.randn(T, h, D, device="cuda").bfloat16() for h in (H, Hkv))
    freq, _ = tt.rotary_frequencies(D)
    check(tt, q, k, torch.arange(T, dtype=torch.int32, device="cuda"), freq)


def test_strides_alignment_and_repeats(tt):
    S, H, Hkv, D = 53, 6, 2, 64
    freq, axes = tt.rotary_frequencies(D, sections=(16, 8, 8))
    pos = torch.randint(0, 5000, (3, S), device="cuda", dtype=torch.int32)
    rows = torch.randn(S, H + 2 * Hkv, D, device="cuda").bfloat16()       # slices of a projection
    check(tt, rows[:, :H], rows[:, H:H + Hkv], pos, freq, axes)
    odd = torch.randn(S, H, D + 1, device="cuda").bfloat16()                # rows off 16 bytes
    check(tt, odd[..., 1:], None, pos, freq, axes)
    off = torch.randn(S * H * D + 1, device="cuda")[1:].view(S, H, D)
    check(tt, off, off[:, :3], pos, freq, axes)
    f1, _ = tt.rotary_frequencies(D)
    many = torch.randn(1, H, S, D, device="cuda").expand(4, H, S, D)        # one batch entry shown four times
    check(tt, many, None, torch.randint(0, 5000, (1, 4, S), device="cuda", dtype=torch.int32), f1)
    turned = torch.randn(S, H, D, device="cuda").transpose(0, 1).contiguous().transpose(0, 1)   # head-major rows
    check(tt, turned, None, pos, freq, axes)
    # a gradient that repeats over the heads
    wq = weights(D, torch.float32, 3)
    g = torch.randn(S, 1, D, device="cuda").expand(S, H, D)
    one = tt.norm_rotary_backward(g, None, off, None, wq, None, pos, freq, axes)
    two = tt.norm_rotary_backward(g.contiguous(), None, off, None, wq, None, pos, freq, axes)
    assert torch.equal(one[0], two[0]) and torch.equal(one[2], two[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R", [64, 24])
def test_in_place_and_into_slices(tt, dtype, R):
    S, H, Hkv, D = 41, 4, 2, 64
    freq, axes = tt.rotary_frequencies(R)
    pos = torch.arange(S, dtype=torch.int32, device="cuda") * 77
    rows = torch.randn(S, H + 2 * Hkv, D, device="cuda").to(dtype)
    q, k, wq, wk = rows[:, :H], rows[:, H:H + Hkv], weights(D, dtype, 1), weights(D, dtype, 2)
    want = tt.norm_rotary_forward(q, k, wq, wk, pos, freq)
    other = torch.full_like(rows, 7.0)
    tt.norm_rotary_forward(q, k, wq, wk, pos, freq, out_q=other[:, :H], out_k=other[:, H:H + Hkv])
    assert torch.equal(other[:, :H], want[0]) and torch.equal(other[:, H:H + Hkv], want[1]) and bool((other[:, H + Hkv:] == 7).all())
    g = torch.randn_like(rows)
    back = tt.norm_rotary_backward(g[:, :H], g[:, H:H + Hkv], q, k, wq, wk, pos, freq)
    kept = g[:, H + Hkv:].clone()
    got = tt.norm_rotary_backward(g[:, :H], g[:, H:H + Hkv], q, k, wq, wk, pos, freq, out_q=g[:, :H], out_k=g[:, H:H + Hkv])
    assert all(torch.equal(a, b) for a, b in zip(got, back)) and torch.equal(g[:, H + Hkv:], kept)
    values = rows[:, H + Hkv:].clone()
    got = tt.norm_rotary_forward(q, k, wq, wk, pos, freq, out_q=q, out_k=k)
    assert got[0] is q or got[0].data_ptr() == q.data_ptr()
    assert torch.equal(rows[:, :H], want[0]) and torch.equal(rows[:, H:H + Hkv], want[1]) and torch.equal(rows[:, H + Hkv:], values)


def test_rows_of_zeros_and_extremes(tt):
    """A row of zeros gives zeros, rows of very small and very large values their unit; NaN stays in its row."""
    D = 128
    x = torch.randn(6, 2, D, device="cuda")
    x[0] = 0
    x[1] *= 1e-12
    x[2] *= 1e15
    x[3, 0, 5] = float("nan")
    w = torch.ones(D, device="cuda")
    freq, _ = tt.rotary_frequencies(D)
    pos = torch.arange(6, dtype=torch.int32, device="cuda")
    y, _ = tt.norm_rotary_forward(x, None, w, None, pos, freq)
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[3, 0]).all()) and not bool(torch.isnan(y[3, 1]).any())
    for row in (1, 2, 4):
        near(y[row], *nr.forward(host(x[row]), host(w), nr.angles(np.array([[row]]), freq.tolist(), None)))
    g = torch.randn_like(x)
    dx, _, dw, _ = tt.norm_rotary_backward(g, None, x, None, w, None, pos, freq)
    dx0, bound, _, _ = nr.backward(host(g[0]), host(x[0]), host(w), nr.angles(np.array([[0]]), freq.tolist(), None))
    near(dx[0], dx0, bound)
    assert bool(torch.isnan(dw).any()) and not bool(torch.isnan(dx[4]).any())


def test_no_rows(tt):
    freq, _ = tt.rotary_frequencies(64)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    q, k = (torch.zeros(0, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    pos = torch.zeros(0, dtype=torch.int32, device="cuda")
    a, b = tt.norm_rotary_forward(q, k, w, w, pos, freq)
    assert a.shape == q.shape and b.shape == k.shape
    got = tt.norm_rotary_backward(q, k, q, k, w, w, pos, freq)
    assert bool((got[2] == 0).all()) and bool((got[3] == 0).all())


def test_gradient_against_differences(tt):
    """The kernel's gradients along a direction against central differences of the formula in 64 bits: the difference is off by
    h^2 / 6 of the third derivative, which for these sizes is far below the gradients' own bound, taken as 1e-4 of the sum of magnitudes."""
    T, H, D, R, h = 5, 2, 32, 16, 1e-5
    rng = np.random.default_rng(4)
    x, w, c = rng.standard_normal((T, H, D)), 1 + 0.3 * rng.standard_normal(D), rng.standard_normal((T, H, D))
    to = lambda a: torch.from_numpy(a).float().cuda()
    x, w, c = (host(to(a)) for a in (x, w, c))
    freq, _ = tt.rotary_frequencies(R)
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 13
    t = angles(pos, freq, None, False)
    dx, _, dw, _ = tt.norm_rotary_backward(to(c), None, to(x), None, to(w), None, pos, freq, interleaved=True, scale=1.5)
    loss = lambda x, w: (nr.forward(x, w, t, True, 1.5)[0] * c).sum()
    for seed in range(3):
        e, f = np.random.default_rng(seed).standard_normal(x.shape), np.random.default_rng(seed + 9).standard_normal(D)
        got = (host(dx) * e).sum()
        assert abs(got - (loss(x + h * e, w) - loss(x - h * e, w)) / (2 * h)) <= 1e-4 * np.abs(host(dx) * e).sum()
        got = (host(dw) * f).sum()
        assert abs(got - (loss(x, w + h * f) - loss(x, w - h * f)) / (2 * h)) <= 1e-4 * np.abs(host(dw) * f).sum()


def test_other_streams_and_graphs(tt):
    T, H, Hkv, D = 70, 8, 2, 128
    q, k = (torch.randn(T, h, D, device="cuda").bfloat16() for h in (H, Hkv))
    g = torch.randn_like(q), torch.randn_like(k)
    w = weights(D, torch.float32, 1)
    freq, _ = tt.rotary_frequencies(D)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    want = tt.norm_rotary_forward(q, k, w, w, pos, freq) + tt.norm_rotary_backward(*g, q, k, w, w, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tt.norm_rotary_forward(q, k, w, w, pos, freq) + tt.norm_rotary_backward(*g, q, k, w, w, pos, freq)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tt.norm_rotary_forward(q, k, w, w, pos, freq) + tt.norm_rotary_backward(*g, q, k, w, w, pos, freq)
    old = [x.clone() for x in (q, *g)]
    q.normal_(), g[0].normal_()
    graph.replay()
    want = tt.norm_rotary_forward(q, k, w, w, pos, freq) + tt.norm_rotary_backward(*g, q, k, w, w, pos, freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not torch.equal(q, old[0])


def test_refusals(tt):
    q, k = torch.randn(5, 4, 64, device="cuda"), torch.randn(5, 2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    freq, _ = tt.rotary_frequencies(64)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    fwd = lambda **kw: tt.norm_rotary_forward(**{**dict(q=q, k=k, q_weight=w, k_weight=w, positions=pos, inv_freq=freq), **kw})
    back = lambda **kw: tt.norm_rotary_backward(**{**dict(dq=q, dk=k, q=q + 1, k=k + 1, q_weight=w, k_weight=w, positions=pos, inv_freq=freq), **kw})
    for call in (fwd, back):
        for bad in (dict(q_weight=None), dict(k_weight=None), dict(q_weight=w[:32]), dict(q_weight=w.double()), dict(q_weight=w.bfloat16()), dict(q_weight=w.cpu()),
                    dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=None), dict(positions=pos[:4]), dict(inv_freq=freq.float()),
                    dict(positions=pos.long()), dict(k=None), dict(scale=float("nan")), dict(out_q=torch.empty(5, 4, 32, device="cuda")),
                    dict(q=q.cpu()), dict(k=k.bfloat16()), dict(axes=torch.zeros(3, dtype=torch.int32, device="cuda"))):
            with pytest.raises(ValueError):
                call(**bad)
    x = q + 1
    with pytest.raises(ValueError):
        back(q=x, out_q=x)              # the gradient onto the input
    with pytest.raises(ValueError):
        back(q=q, out_q=q)              # ... or where the upstream gradient is the input
    with pytest.raises(ValueError):
        back(workspace=torch.empty(3, device="cpu"))
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    back(workspace=small)               # too small: another is made


def test_strides_beyond_32_bits(tt):
    T, H, D, far = 3, 2, 64, 1_200_000_000
    base = torch.empty(2 * far + H * D, device="cuda", dtype=torch.bfloat16)
    x = base.as_strided((T, H, D), (far, D, 1))
    x.copy_(torch.randn(T, H, D, device="cuda"))
    freq, _ = tt.rotary_frequencies(D)
    pos, w = torch.arange(T, dtype=torch.int32, device="cuda"), weights(D, torch.float32, 4)
    near_by = x.contiguous()
    want, _ = tt.norm_rotary_forward(near_by, None, w, None, pos, freq)
    assert torch.equal(tt.norm_rotary_forward(x, None, w, None, pos, freq)[0], want)
    g = torch.randn_like(near_by)
    a, b = (tt.norm_rotary_backward(g, None, y, None, w, None, pos, freq) for y in (x, near_by))
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    got, _ = tt.norm_rotary_forward(near_by, None, w, None, pos, freq, out_q=x)
    assert got is x and torch.equal(x, want)


def test_neighbouring_memory(tt):
    """Outputs and workspace end where they end."""
    import ctypes

    from test_gpu_canary import Guarded
    for T, H, Hkv, D, R, dtype in ((1, 1, 1, 64, 64, torch.bfloat16), (37, 5, 2, 80, 40, torch.bfloat16), (9, 3, 1, 50, 18, torch.float32), (600, 8, 2, 128, 128, torch.bfloat16)):
        q, k = (torch.randn(T, h, D, device="cuda").to(dtype) for h in (H, Hkv))
        freq, _ = tt.rotary_frequencies(R)
        pos, w = torch.arange(T, dtype=torch.int32, device="cuda"), weights(D, torch.float32, 5)
        d = tt.capi.RotaryDesc(B=1, S=T, H=H, Hkv=Hkv, D=D, R=R, n_axes=1, dtype=tt.capi.TT_F32, interleaved=0, scale=1.0)
        need = int(tt.capi.lib.tt_norm_rotary_bwd_workspace_bytes(ctypes.byref(d)))
        assert need > 0
        a, b, ws = Guarded((T, H, D), dtype), Guarded((T, Hkv, D), dtype), Guarded((need,), torch.uint8)
        want = tt.norm_rotary_forward(q, k, w, w, pos, freq)
        tt.norm_rotary_forward(q, k, w, w, pos, freq, out_q=a.t, out_k=b.t)
        torch.cuda.synchronize()
        assert a.intact() and b.intact() and torch.equal(a.t, want[0]) and torch.equal(b.t, want[1])
        want = tt.norm_rotary_backward(q, k, q + 1, k + 1, w, w, pos, freq)
        got = tt.norm_rotary_backward(q, k, q + 1, k + 1, w, w, pos, freq, out_q=a.t, out_k=b.t, workspace=ws.t)
        torch.cuda.synchronize()
        assert a.intact() and b.intact() and ws.intact() and all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("H,Hkv", [(1, 40), (64, 1), (7, 3)])
def test_shares_of_the_gradient_s_ctas(tt, H, Hkv):
    """Tensors of very different numbers of heads, and many more tokens than CTAs."""
    T, D = 2500, 64
    q, k = (torch.randn(T, h, D, device="cuda") for h in (H, Hkv))
    freq, _ = tt.rotary_frequencies(D)
    check(tt, q, k, torch.arange(T, dtype=torch.int32, device="cuda"), freq)
