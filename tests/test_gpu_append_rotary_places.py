"""Appending to the paged 16-bit cache from and to every place that the call takes: with and without queries at every access width, and pools
that start anywhere.  Checks and bounds are those of test_gpu_append_rotary."""
import pytest

from test_gpu_append_rotary import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("layout", ["fused", "apart", "odd"])
def test_keys_without_queries(tt, layout, normed, dtype):
    """Rows of 16 bytes and of single elements, whole rows with two units to a lane and rows of a narrower rotation."""
    for T, Hkv, D, R, page, interleaved in ((1, 1, 64, 64, 16, False), (70, 8, 128, 128, 64, False), (33, 3, 64, 64, 48, True), (45, 2, 128, 20, 7, False), (300, 1, 128, 2, 16, True)):
        c = Case(tt, T, 2, Hkv, D, R, page, T // page + 2, dtype, normed, seed=T, layout=layout)
        c.check(tt, interleaved=interleaved, with_q=False)
        c.check(tt, interleaved=interleaved, with_q=False, with_k=True)


def at_byte(p, off):
    """A copy of a pool that starts `off` bytes behind a multiple of 256, with guards around it."""
    n = p.numel()
    whole = torch.full((n + 256,), 9.0, device="cuda", dtype=p.dtype)
    assert whole.data_ptr() % 256 == 0
    view = whole[64 + off // 2:64 + off // 2 + n].view(p.shape)
    view.copy_(p)
    return whole, view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("with_q", [False, True])
@pytest.mark.parametrize("k_off,v_off", [(2, 0), (0, 2), (8, 0), (0, 8), (4, 8), (2, 2), (14, 6)])
def test_pools_that_start_anywhere(tt, k_off, v_off, with_q, normed, dtype):
    """Pools need to be multiples of their element size only: each is written as one on 16 bytes is, and nothing around it.  (The sum of a row's squares
    depends on the accesses' width, so the values are held to the bounds.)"""
    for T, H, Hkv, D, R, page in ((1, 4, 1, 64, 64, 16), (90, 8, 2, 128, 128, 16), (40, 2, 3, 64, 32, 48)):
        c = Case(tt, T, H, Hkv, D, R, page, T // page + 2, dtype, normed, seed=T, layout="apart")
        wholes, c.pools = zip(*(at_byte(p, off) for p, off in zip(c.pools, (k_off, v_off))))
        assert [p.data_ptr() % 16 for p in c.pools] == [k_off, v_off] and all(p.is_contiguous() for p in c.pools)
        c.check(tt, with_q=with_q)
        c.check(tt, with_q=with_q, with_k=True)
        for whole, pool, off in zip(wholes, c.pools, (k_off, v_off)):
            first = 64 + off // 2
            assert bool((whole[:first] == 9).all()) and bool((whole[first + pool.numel():] == 9).all())
