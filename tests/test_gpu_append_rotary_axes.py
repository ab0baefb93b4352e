"""Appending to the paged 16-bit cache with positions on several axes, and beside the separate calls.  Bounds are those of norm_rotary_oracle."""
import numpy as np
import pytest

import norm_rotary_oracle as nr
from test_gpu_append_rotary import Case, host, near

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("T,H,Hkv,D,R,A,cyclic", [(1, 4, 1, 64, 64, 2, False), (90, 8, 2, 128, 128, 3, False), (33, 3, 3, 64, 24, 4, True), (700, 0, 2, 128, 64, 3, True), (50, 5, 1, 64, 64, 1, False)])
def test_axes(tt, T, H, Hkv, D, R, A, cyclic, normed, dtype):
    for layout in ("fused", "apart", "odd"):
        for interleaved in (False, True):
            c = Case(tt, T, max(H, 1), Hkv, D, R, 16, T // 16 + 2, dtype, normed, seed=T, layout=layout)
            sections = [R // 2 // A + (a < R // 2 % A) for a in range(A)]
            freq, axes = tt.rotary_frequencies(R, sections=sections, cyclic=cyclic)
            axes = torch.zeros(R // 2, dtype=torch.int32, device="cuda") if axes is None else axes
            wide = torch.from_numpy(c.rng.integers(0, 100000, (A, T + 3)).astype(np.int32)).cuda()
            also = torch.empty(T, Hkv, D, device="cuda", dtype=torch.bfloat16)
            t = nr.angles(wide[:, 2:T + 2].cpu().numpy(), freq.tolist(), axes.tolist())[:, None]
            w = [None if x is None else host(x) for x in c.w]
            # rows of positions that lie apart
            got = c.call(tt, positions=wide[:, 2:T + 2], inv_freq=freq, axes=axes, interleaved=interleaved, out_k=also, **({} if H else dict(q=None)))
            assert (got is None) == (H == 0)
            if H:
                near(got, *nr.forward(host(c.q), w[0], t, interleaved))
            near(also, *nr.forward(host(c.k), w[1], t, interleaved))
            at = c.slots.long()
            assert torch.equal(c.pools[0][at // 16, :, at % 16], also) and torch.equal(c.pools[1][at // 16, :, at % 16], c.v.bfloat16())


def test_axes_that_no_row_has(tt):
    """Axes beyond the positions' rows count as the nearest, as in the separate calls; one row without axes is all pairs'."""
    c = Case(tt, 40, 4, 2, 64, 64, 16, 4, normed=True, seed=2)
    pos = torch.stack((c.pos, c.pos.flip(0)))
    axes = torch.tensor([-5, 0, 1, 7] * 8, dtype=torch.int32, device="cuda")
    want = c.call(tt, positions=pos, axes=axes.clamp(0, 1)).clone()
    pools = [p.clone() for p in c.pools]
    assert torch.equal(c.call(tt, positions=pos, axes=axes), want) and all(torch.equal(a, b) for a, b in zip(pools, c.pools))
    want = c.call(tt).clone()
    assert torch.equal(c.call(tt, positions=c.pos[None]), want)
    for bad in (dict(positions=pos), dict(positions=pos, axes=axes[:5]), dict(positions=pos, axes=axes.long()), dict(positions=pos[:, :7], axes=axes), dict(positions=pos.t().contiguous(), axes=axes)):
        with pytest.raises(ValueError):
            c.call(tt, **bad)


@pytest.mark.parametrize("layout", ["fused", "apart", "odd"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D,R,interleaved", [(4, 2, 64, 64, False), (32, 8, 128, 128, False), (8, 2, 128, 128, True), (32, 4, 64, 16, True), (6, 3, 128, 60, False), (2, 1, 64, 8, True)])
def test_as_the_norm_and_a_copy(tt, H, Hkv, D, R, interleaved, dtype, layout):
    """Where the values and the pools lie at multiples of what queries and keys do, accesses are of one width, and queries and keys are those of
    `norm_rotary_forward` to the bit (of floats, once rounded)."""
    c = Case(tt, 150, H, Hkv, D, R, 16, 12, dtype, True, seed=2, layout=layout)
    got = c.call(tt, interleaved=interleaved)
    q, k = tt.norm_rotary_forward(c.q, c.k, *c.w, c.pos, c.freq, interleaved=interleaved)
    at = c.slots.long()
    assert torch.equal(got, q.bfloat16()) and torch.equal(c.pools[0][at // 16, :, at % 16], k.bfloat16())
