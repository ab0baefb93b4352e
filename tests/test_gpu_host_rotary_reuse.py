"""One `Rotary` op applied to several inputs: each one's gradient is of its own head dim, type and place."""
import importlib

import numpy as np
import pytest

from test_gpu_host_rotary import turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def opt(tt):
    return importlib.import_module("pku-aiprogramming_b200.optimizer")


def test_two_head_dims_one_op(opt):
    """Both orders of the backward passes; the bound is that of one op for each."""
    rng = np.random.default_rng(0)
    S = 9
    pos = rng.integers(0, 300, S)
    for order in ((0, 1), (1, 0)):
        turn = opt.Rotary(pos)
        data = [(rng.standard_normal((1, 2, S, D)).astype(np.float32), rng.standard_normal((1, 2, S, D)).astype(np.float32)) for D in (32, 16)]
        xs = [opt.Tensor(x) for x, _ in data]
        ys = [turn(x) for x in xs]
        for i in order:
            x, y, (x0, g0) = xs[i], ys[i], data[i]
            y.backward(opt.Tensor(g0, requires_grad=False))
            freq, axes, _ = opt.rotary_table(x0.shape[-1])
            assert np.abs(y.numpy() - turned(x0, pos[None], freq, axes)).max() < 1e-6 * 2 * np.abs(x0).max()
            assert np.abs(x.grad.numpy() - turned(g0, pos[None], freq, axes, back=True)).max() < 1e-6 * 2 * np.abs(g0).max()


def test_types_and_places_one_op(opt):
    """Resident bf16, resident float and NumPy inputs through one op, backward in every order."""
    import itertools
    rng = np.random.default_rng(1)
    S, D = 5, 8
    pos = np.stack([rng.integers(0, 300, S), rng.integers(0, 300, S)])
    x0, g0 = (rng.integers(-8, 9, (1, 1, S, D)).astype(np.float32) / 4 for _ in range(2))   # exact in bf16
    freq, axes, _ = opt.rotary_table(D, sections=(1, 3))
    want = turned(g0, pos, freq, axes, back=True)
    for order in itertools.permutations(range(3)):
        turn = opt.Rotary(pos, sections=(1, 3))
        xs = [opt.Tensor(x0, device="gpu", dtype="bfloat16"), opt.Tensor(x0, device="gpu"), opt.Tensor(x0)]
        gs = [opt.Tensor(g0, device="gpu", dtype="bfloat16", requires_grad=False), opt.Tensor(g0, device="gpu", requires_grad=False), opt.Tensor(g0, requires_grad=False)]
        ys = [turn(x) for x in xs]
        for i in order:
            ys[i].backward(gs[i])
            grad = xs[i].grad
            assert grad.is_device == (i < 2) and ys[i].is_device == (i < 2)
            if i < 2:
                assert type(grad.realize_cached_data()) is type(xs[i].realize_cached_data())
            # 1e-6 of |g1| + |g2|, and bf16's half step of the value
            assert (np.abs(grad.numpy() - want) <= 1e-6 * 2 * np.abs(g0).max() + (2.0 ** -8 * np.abs(want) if i == 0 else 0)).all()
