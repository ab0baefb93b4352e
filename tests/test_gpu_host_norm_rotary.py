"""The `NormRotary` autograd op and `myLayer.NormRotaryForward/Backward`: through Python, pybind and C++ to the kernels; bounds as in
norm_rotary_oracle."""
import importlib
import os
import sys

import numpy as np
import pytest

import norm_rotary_oracle as nr

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def opt(tt):
    return importlib.import_module("pku-aiprogramming_b200.optimizer")


@pytest.fixture(scope="module")
def mods(tt):
    sys.path.insert(0, os.path.join(ROOT, "pku-aiprogramming_b200", "host_modules"))
    import myLayer
    import myTensor
    return myTensor, myLayer


def near(got, want, bound, eps=2.0 ** -23):
    ok, worst = nr.within(got.astype(np.float64), want, bound, eps)
    assert ok, worst


def angles(pos, freq, axes):
    t = nr.angles(pos, freq, axes)
    return t if t.ndim == 2 else t[:, None]


@pytest.mark.parametrize("interleaved", [False, True])
def test_op_and_gradients(opt, interleaved):
    rng = np.random.default_rng(0)
    B, H, S, D = 2, 3, 17, 40
    x0, g0 = (rng.standard_normal((B, H, S, D)).astype(np.float32) for _ in range(2))
    w0 = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    for pos, sections in ((rng.integers(0, 5000, S), None), (rng.integers(0, 5000, (2, S)), (4, 6)), (rng.integers(0, 5000, (2, B, S)), (4, 6))):
        freq, axes, _ = opt.rotary_table(20, sections=sections)
        t = angles(pos.reshape((1,) * (2 - pos.ndim) + pos.shape), freq, axes)
        x, w = opt.Tensor(x0), opt.Tensor(w0)
        y = opt.norm_rotary(x, w, pos, eps=1e-3, rotary_dim=20, sections=sections, interleaved=interleaved, scale=1.25)
        y.backward(opt.Tensor(g0, requires_grad=False))
        near(y.numpy(), *nr.forward(x0, w0.astype(np.float64), t, interleaved, 1.25, 1e-3))
        dx, edx, dw, edw = nr.backward(g0, x0, w0.astype(np.float64), t, interleaved, 1.25, 1e-3)
        near(x.grad.numpy(), dx, edx)
        near(w.grad.numpy(), dw, edw)
        assert y.numpy().dtype == x.grad.numpy().dtype == w.grad.numpy().dtype == np.float32


def test_one_op_on_several_inputs(opt):
    """Queries and keys of one step, each with its weight, by one op: each gradient is of its own input."""
    rng = np.random.default_rng(1)
    S, pos = 9, np.arange(9) * 5
    op = opt.NormRotary(pos)
    xs = [rng.standard_normal((1, h, S, D)).astype(np.float32) for h, D in ((4, 16), (2, 16), (3, 8))]
    ws = [(1 + 0.2 * rng.standard_normal(x.shape[-1])).astype(np.float32) for x in xs]
    nodes = [(opt.Tensor(x), opt.Tensor(w)) for x, w in zip(xs, ws)]
    ys = [op(x, w) for x, w in nodes]
    for i in (1, 2, 0):
        g0 = rng.standard_normal(xs[i].shape).astype(np.float32)
        gx, gw = ys[i].op.gradient_as_tuple(opt.Tensor(g0, requires_grad=False), ys[i])
        freq, axes, _ = opt.rotary_table(xs[i].shape[-1])
        dx, edx, dw, edw = nr.backward(g0, xs[i], ws[i].astype(np.float64), angles(pos[None], freq, axes))
        near(gx.numpy(), dx, edx)
        near(gw.numpy(), dw, edw)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_in_front_of_attention(opt, oracle, dtype):
    """Gradients of attention(norm_rotary(q), norm_rotary(k), v), device-resident, against the oracle's with q and k normed and turned in NumPy."""
    B, H, S, D = 1, 2, 40, 64
    q0, k0, v0, g0 = (oracle.bf16_round(x) for x in oracle.make_inputs(5, B, H, S, S, D))
    rng = np.random.default_rng(2)
    wq, wk = (oracle.bf16_round((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2))
    pos = np.arange(S)
    freq, axes, _ = opt.rotary_table(D)
    t = angles(pos[None], freq, axes)
    q, k, v, a, b = (opt.Tensor(x, device="gpu", dtype=dtype) for x in (q0, k0, v0, wq, wk))
    norm = lambda x, w: opt.norm_rotary(x, w, pos, dtype=dtype)
    out = opt.attention(norm(q, a), norm(k, b), v, causal=True, dtype=dtype)
    out.backward(opt.Tensor(g0, device="gpu", dtype=dtype, requires_grad=False))
    qr, kr = (nr.forward(x, w.astype(np.float64), t)[0].astype(np.float32) for x, w in ((q0, wq), (k0, wk)))
    if dtype == "bfloat16":
        qr, kr = oracle.bf16_round(qr), oracle.bf16_round(kr)
    o, _, dq, dk, dv = oracle.attention_backward(qr, kr, v0, g0, True)
    e = 2e-2   # the bf16 attention's bound; a turn back makes at most sqrt(2) of it in a channel
    pairs = [(out, o, e), (v.grad, dv, oracle.bf16_grad_tol(dv))]
    for got_x, got_w, dz, x, w in ((q.grad, a.grad, dq, q0, wq), (k.grad, b.grad, dk, k0, wk)):
        x, w = x.astype(np.float64), w.astype(np.float64)
        dx, _, dw, _ = nr.backward(dz, x, w, t)
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
        off = 1.5 * (oracle.bf16_grad_tol(dz) + 2.0 ** -8 * np.abs(dz).max())   # (and its rounding to bf16 between the two ops)
        pairs.append((got_x, dx, r * (np.abs(w) + np.abs(x) * (np.abs(w * x)).mean(-1, keepdims=True) * r * r) * off + 2.0 ** -8 * np.abs(dx)))
        pairs.append((got_w, dw, (np.abs(x * r) * off).reshape(-1, D).sum(0) + 2.0 ** -8 * np.abs(dw)))
    for got, ref, room in pairs:
        assert got.is_device
        if dtype == "float32":
            assert oracle.rel_err(got.numpy(), ref) <= 1e-5
        else:
            assert (np.abs(got.numpy() - ref) <= room).all()


def test_layer_functions_and_refusals(opt, mods):
    mt, ml = mods
    rng = np.random.default_rng(1)
    x0 = rng.standard_normal((1, 2, 5, 8)).astype(np.float32)
    up = lambda a: mt.Tensor_float(np.ascontiguousarray(a, np.float32), "gpu")
    x, w, y, gx, gw = up(x0), up(np.ones(8)), up(np.ones(1)), up(np.ones(1)), up(np.ones(1))
    pos, freq, axes = mt.Tensor_int(np.arange(5, dtype=np.int32).reshape(1, 5), "gpu"), mt.Tensor_double(np.ones(4), "gpu"), mt.Tensor_int(np.zeros(4, np.int32), "gpu")
    rest = (pos, freq, axes)
    ml.NormRotaryForward(x, w, y, *rest)
    ml.NormRotaryBackward(x, w, y, gx, gw, *rest)
    first = gx.numpy().copy()
    ml.NormRotaryBackward(x, w, y, y, gw, *rest)      # onto the upstream gradient
    assert np.array_equal(y.numpy(), first)
    for bad in ((mt.Tensor_float(x0, "cpu"), w), (x, mt.Tensor_float(np.ones(8, np.float32), "cpu")), (x, up(np.ones(7))), (x, up(np.ones((1, 8)))), (up(x0[0]), w)):
        with pytest.raises(ValueError):
            ml.NormRotaryForward(*bad, gx, *rest)
        with pytest.raises(ValueError):
            ml.NormRotaryBackward(*bad, up(x0), gx, gw, *rest)
    for call in (lambda: ml.NormRotaryForward(x, w, gx, *rest, eps=0.0), lambda: ml.NormRotaryBackward(x, w, up(x0[:, :1]), gx, gw, *rest), lambda: ml.NormRotaryBackward(x, w, up(x0), x, gw, *rest),
                 lambda: ml.NormRotaryBackward(x, w, up(x0), gx, w, *rest), lambda: opt.NormRotary(np.arange(5), eps=0.0), lambda: opt.NormRotary(np.arange(5), eps=float("nan")),
                 lambda: opt.norm_rotary(opt.Tensor(x0), opt.Tensor(np.ones(7, np.float32)), np.arange(5))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        opt.norm_rotary(opt.Tensor(x0, device="gpu"), opt.Tensor(np.ones(8, np.float32)), np.arange(5))
    with pytest.raises(TypeError):
        opt.norm_rotary(opt.Tensor(x0, device="gpu"), opt.Tensor(np.ones(8, np.float32), device="gpu", dtype="bfloat16"), np.arange(5))
