"""Decode over the 4-bit cache with queries of every finite size: the head's largest value anywhere in bf16's range, scores moderate, vanishing or far beyond
what the exponential tells apart."""
import numpy as np
import pytest

from test_gpu_decode_q4 import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [90, 109, 111, 112, 113, 118, 125, -90, -101, -115, -125])
@pytest.mark.parametrize("H,hkv,D", [(4, 2, 128), (12, 1, 64)])
def test_large_and_small_queries_with_moderate_scores(tt, power, H, hkv, D):
    """`scale` takes back what q is larger or smaller by (within the floats that have all their bits); the bounds are those of ordinary queries."""
    scale = 2.0 ** max(-power, -120) * D ** -0.5 if power > 0 else 2.0 ** min(-power, 120) * D ** -0.5
    c = Case([300, 40, 1, 0], H, hkv, D, 16, q_scale=2.0 ** power)
    c.check(*tt.attention_decode_q4(**c.args(), scale=scale), scale)


@pytest.mark.parametrize("power,scale", [(-100, 2.0 ** -60), (-110, 2.0 ** -30), (-126, 2.0 ** -100), (0, 2.0 ** -140)])
def test_scores_that_vanish(tt, power, scale):
    """q and scale both small: all keys count alike, and the places behind the last one do not."""
    c = Case([300, 41, 7, 0], 4, 2, 64, 16, q_scale=2.0 ** power)
    c.check(*tt.attention_decode_q4(**c.args(), scale=scale), scale)


@pytest.mark.parametrize("power", [0, 60, 110, 112, 120, 126])
@pytest.mark.parametrize("G", [1, 3, 16])
def test_one_key_far_above_the_others(tt, power, G):
    """Scores of up to 2^126: the result is that key's values, exactly, and the log-sum-exp its score.  Keys differ by a factor of two from
    one to the next in the only channel that q has, so a score is one exact product times scale and log2 e, and the log-sum-exp that times ln 2: eight
    roundings of 2^-24 with those of the three constants."""
    D, page, n = 128, 16, 23
    c = Case([n, 600], G, 1, D, page)
    rng = np.random.default_rng(3)
    k = np.zeros((n, 1, D))
    k[:, 0, 5] = 2.0 ** (rng.permutation(n) - 19)   # 2^-19 .. 2^3
    slots = c.table[0, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
    c.pools[0].write(slots, k)
    q = torch.zeros(2, G, 1, D)
    q[0, :, 0, 5] = 2.0 ** power * (1 + torch.arange(G) / 16)
    c.q = q.bfloat16()
    out, lse = tt.attention_decode_q4(**c.args())
    if power == 0:   # the others count, too
        c.check(out, lse)
        return
    kept, values = c.rows(0)
    best = int(kept[:, 0, 5].argmax())
    want = c.q[0, :, 0, 5].double().numpy() * kept[best, 0, 5] * D ** -0.5
    assert (np.abs(lse[0, :, 0].double().cpu().numpy() - want) <= 2.0 ** -21 * want).all()
    assert np.array_equal(out[0, :, 0].double().cpu().numpy(), np.broadcast_to(values[best, 0], (G, D)))


@pytest.mark.parametrize("power", [18, 20, 22, 24, 26, 30, 60, 115])
@pytest.mark.parametrize("G,D,n", [(4, 128, 2000), (12, 64, 700), (2, 64, 90)])
def test_scores_beyond_the_exponents_range(tt, power, G, D, n):
    """Random keys and queries of 2^power: scores whose own last bit is more than one.  The largest is ahead of the others by more than a score may be
    off -- (D + 4) 2^-23 of sum |q k|, the bound of ordinary queries and the product's rounding -- so the result is its key's values."""
    c = Case([n], G, 1, D, 16, seed=G, q_scale=2.0 ** power)
    k, v = (x[:, 0] for x in c.rows(0))
    q = c.q[0, :, 0].double().numpy()
    s = q @ k.T * D ** -0.5
    off = (D + 4) * 2.0 ** -23 * (np.abs(q) @ np.abs(k).T).max(-1) * D ** -0.5
    two = np.sort(s, -1)[:, -2:]
    sure = two[:, 1] - two[:, 0] > 2 * off + 60   # (60: nothing left of the second in the sum)
    out, lse = tt.attention_decode_q4(**c.args())
    assert sure.any()
    want = v[s.argmax(-1)]
    assert np.array_equal(out[0, :, 0].double().cpu().numpy()[sure], want[sure])
    assert (np.abs(lse[0, :, 0].double().cpu().numpy() - two[:, 1]) <= off + 2.0 ** -20 * np.abs(two[:, 1]))[sure].all()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
