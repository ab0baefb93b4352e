"""The `Rotary` op's bookkeeping, with NumPy in the place of the native modules: one op on several inputs."""
import importlib

import numpy as np
import pytest


class _Base:
    def __init__(self, x, place):
        assert place == "gpu"
        self.x = np.zeros(x, self.kind) if isinstance(x, list) else np.array(x, self.kind)

    def get_device(self):
        return "gpu"

    def get_shape(self):
        return list(self.x.shape)

    def get_data(self):
        return self.x.reshape(-1).tolist()

    def numpy(self):
        return self.x


class Tensor_float(_Base):
    kind = np.float32


class Tensor_bf16(_Base):
    kind = np.float32


class Tensor_int(_Base):
    kind = np.int32


class Tensor_double(_Base):
    kind = np.float64


class _Layers:
    @staticmethod
    def _turn(T, sign):
        def call(x, y, pos, freq, axes, interleaved, scale):
            assert type(x) is T and type(y) is T and not interleaved
            n, out = len(freq.x), x.x.astype(np.float64).copy()
            assert 2 * n <= x.x.shape[-1]
            for i in range(n):
                t = pos.x[axes.x[i]] * freq.x[i]
                a, b = x.x[..., i].astype(np.float64), x.x[..., i + n].astype(np.float64)
                out[..., i], out[..., i + n] = (a * np.cos(t) - sign * b * np.sin(t)) * scale, (b * np.cos(t) + sign * a * np.sin(t)) * scale
            y.x = out.astype(np.float32)
        return staticmethod(call)

    RotaryForward, RotaryBackward = _turn.__func__(Tensor_float, 1), _turn.__func__(Tensor_float, -1)
    RotaryForward_bf16, RotaryBackward_bf16 = _turn.__func__(Tensor_bf16, 1), _turn.__func__(Tensor_bf16, -1)


class _Tensors:
    Tensor_float, Tensor_bf16, Tensor_int, Tensor_double = Tensor_float, Tensor_bf16, Tensor_int, Tensor_double


@pytest.fixture
def opt(tt, monkeypatch):
    ops = importlib.import_module("pku-aiprogramming_b200.optimizer.operators")
    monkeypatch.setattr(ops, "_native", lambda: (_Tensors, _Layers))
    return ops


def _gradient(opt, make, x, g):
    """By an op of its own."""
    return _leaf_gradient(opt, make()(x), x, g)


def _leaf_gradient(opt, y, x, g):
    (grad,) = y.op.gradient_as_tuple(g, y)
    return grad


def test_head_dims(opt):
    rng = np.random.default_rng(0)
    pos = rng.integers(0, 50, 6)
    xs = [opt.Tensor(rng.standard_normal((1, 2, 6, D)).astype(np.float32)) for D in (16, 8, 32)]
    gs = [opt.Tensor(rng.standard_normal(x.shape).astype(np.float32), requires_grad=False) for x in xs]
    turn = opt.Rotary(pos)
    ys = [turn(x) for x in xs]
    for i in (0, 2, 1, 0):
        want = _gradient(opt, lambda: opt.Rotary(pos), xs[i], gs[i]).numpy()
        assert np.array_equal(_leaf_gradient(opt, ys[i], xs[i], gs[i]).numpy(), want)


def test_types_and_places(opt):
    rng = np.random.default_rng(1)
    pos, x0, g0 = rng.integers(0, 50, 6), rng.standard_normal((1, 2, 6, 8)).astype(np.float32), rng.standard_normal((1, 2, 6, 8)).astype(np.float32)
    nodes = [opt.Tensor.make_const(T(x0, "gpu"), requires_grad=True) for T in (Tensor_bf16, Tensor_float)] + [opt.Tensor(x0), opt.Tensor(x0.astype(np.float64))]
    grads = [opt.Tensor.make_const(T(g0, "gpu")) for T in (Tensor_bf16, Tensor_float)] + [opt.Tensor(g0, requires_grad=False)] * 2
    turn = opt.Rotary(pos)
    ys = [turn(x) for x in nodes]
    for i in (0, 1, 2, 3, 1, 0):
        got = _leaf_gradient(opt, ys[i], nodes[i], grads[i])
        want = _gradient(opt, lambda: opt.Rotary(pos), nodes[i], grads[i])
        assert type(got.realize_cached_data()) is type(want.realize_cached_data()) and np.array_equal(got.numpy(), want.numpy())
        if i >= 2:
            assert got.dtype == nodes[i].dtype


def test_no_uploads_beyond_those_of_the_forward(opt):
    """The backward of an input takes the positions and frequencies that are on the device."""
    made = []

    class Counted(Tensor_int):
        def __init__(self, *a):
            made.append(1)
            super().__init__(*a)

    tensors = type("M", (), dict(Tensor_float=Tensor_float, Tensor_bf16=Tensor_bf16, Tensor_int=Counted, Tensor_double=Tensor_double))
    opt._native = lambda: (tensors, _Layers)
    pos = np.arange(4)
    turn = opt.Rotary(pos)
    xs = [opt.Tensor(np.ones((1, 1, 4, D), np.float32)) for D in (8, 4)]
    ys = [turn(x) for x in xs]
    n = len(made)
    for x, y in zip(xs, ys):
        _leaf_gradient(opt, y, x, opt.Tensor(np.ones(x.shape, np.float32), requires_grad=False))
    assert len(made) == n
