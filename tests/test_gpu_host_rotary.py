"""The `Rotary` autograd op and `myLayer.RotaryForward/Backward`: through Python, pybind and C++ to the kernels."""
import importlib
import os
import sys

import numpy as np
import pytest

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


def turned(x, pos, freq, axes, interleaved=False, scale=1.0, back=False):
    y = x.astype(np.float64).copy()
    n = len(freq)
    for i in range(n):
        t = pos[axes[i]].astype(np.float64) * freq[i]
        t = t[:, None] if t.ndim == 2 else t[None, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        c, s = np.cos(t) * scale, np.sin(t) * scale * (-1 if back else 1)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


@pytest.mark.parametrize("interleaved", [False, True])
def test_op_and_gradient(opt, interleaved):
    rng = np.random.default_rng(0)
    B, H, S, D = 2, 3, 17, 40
    x0, g0 = (rng.standard_normal((B, H, S, D)).astype(np.float32) for _ in range(2))
    for pos, sections in ((rng.integers(0, 5000, S), None), (rng.integers(0, 5000, (2, S)), (4, 6)), (rng.integers(0, 5000, (2, B, S)), (4, 6))):
        freq, axes, _ = opt.rotary_table(20, sections=sections)
        p = pos.reshape((1,) * (2 - pos.ndim) + pos.shape)
        x = opt.Tensor(x0)
        y = opt.rotary(x, pos, rotary_dim=20, sections=sections, interleaved=interleaved, scale=1.25)
        y.backward(opt.Tensor(g0, requires_grad=False))
        # under 1e-6 of |x1| + |x2| times the scale: see the bound of the torch call's tests
        assert np.abs(y.numpy() - turned(x0, p, freq, axes, interleaved, 1.25)).max() < 1e-6 * 1.25 * 2 * np.abs(x0).max()
        assert np.abs(x.grad.numpy() - turned(g0, p, freq, axes, interleaved, 1.25, True)).max() < 1e-6 * 1.25 * 2 * np.abs(g0).max()
        assert y.numpy().dtype == np.float32


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_in_front_of_attention(opt, oracle, dtype):
    """Gradients of attention(rotary(q), rotary(k), v), device-resident, against the oracle's with q and k turned in NumPy."""
    B, H, S, D = 1, 2, 40, 64
    q0, k0, v0, g0 = (oracle.bf16_round(x) for x in oracle.make_inputs(5, B, H, S, S, D))
    pos = np.stack([np.arange(S), np.arange(S) // 8])
    freq, axes, _ = opt.rotary_table(D, sections=(16, 16))
    q, k, v = (opt.Tensor(x, device="gpu", dtype=dtype) for x in (q0, k0, v0))
    turn = lambda t: opt.rotary(t, pos, sections=(16, 16), dtype=dtype)
    out = opt.attention(turn(q), turn(k), v, causal=True, dtype=dtype)
    out.backward(opt.Tensor(g0, device="gpu", dtype=dtype, requires_grad=False))
    qr, kr = (turned(x, pos, freq, axes).astype(np.float32) for x in (q0, k0))
    if dtype == "bfloat16":
        qr, kr = oracle.bf16_round(qr), oracle.bf16_round(kr)
    o, _, dq, dk, dv = oracle.attention_backward(qr, kr, v0, g0, True)
    want = (o, turned(dq, pos, freq, axes, back=True), turned(dk, pos, freq, axes, back=True), dv)
    for got, ref in zip((out, q.grad, k.grad, v.grad), want):
        assert got.is_device
        if dtype == "float32":
            assert oracle.rel_err(got.numpy(), ref) <= 1e-5
        else:
            # the bf16 attention's bound, twice for gradients that are rounded twice
            assert oracle.max_abs_err(got.numpy(), ref) <= 2 * 2e-2


def test_layer_functions_and_refusals(opt, mods):
    mt, ml = mods
    rng = np.random.default_rng(1)
    x0 = rng.standard_normal((1, 2, 5, 8)).astype(np.float32)
    x, y = mt.Tensor_float(x0, "gpu"), mt.Tensor_float([1], "gpu")
    pos, freq, axes = mt.Tensor_int(np.arange(5, dtype=np.int32).reshape(1, 5), "gpu"), mt.Tensor_double(np.ones(4), "gpu"), mt.Tensor_int(np.zeros(4, np.int32), "gpu")
    ml.RotaryForward(x, y, pos, freq, axes)
    ml.RotaryBackward(y, y, pos, freq, axes)     # in place, and back to where it was
    assert np.abs(y.numpy() - x0).max() < 4e-6
    for bad in ((mt.Tensor_float(x0, "cpu"), pos, freq, axes), (mt.Tensor_float(x0[0], "gpu"), pos, freq, axes), (x, mt.Tensor_int(np.zeros((1, 4), np.int32), "gpu"), freq, axes),
                (x, pos, mt.Tensor_double(np.ones(3), "gpu"), axes), (x, pos, mt.Tensor_double(np.ones(5), "gpu"), mt.Tensor_int(np.zeros(5, np.int32), "gpu"))):
        with pytest.raises(ValueError):
            ml.RotaryForward(bad[0], y, *bad[1:])
    for kw in (dict(positions=np.arange(5.0)), dict(positions=np.arange(5), dtype="float16"), dict(positions=np.full(5, 2 ** 31)), dict(positions=np.zeros((1, 1, 1, 5), int))):
        with pytest.raises(ValueError):
            opt.Rotary(**kw)
    with pytest.raises(ValueError):
        opt.rotary(opt.Tensor(x0), np.arange(5), sections=(2, 2))
