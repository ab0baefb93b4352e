"""Decode over the 8-bit cache with queries of every finite size: the head's largest value anywhere in bf16's range, scores moderate, vanishing or far beyond
what the exponential tells apart.  The bounds are those of test_gpu_decode_q8 where nothing else is said."""
import numpy as np
import pytest

from test_gpu_decode_q8 import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [90, 109, 111, 112, 113, 118, 125, -90, -101, -115, -125])
@pytest.mark.parametrize("H,hkv,D", [(4, 2, 128), (12, 1, 64)])
def test_large_and_small_queries_with_moderate_scores(tt, power, H, hkv, D):
    """`scale` takes back what q is larger or smaller by (within the floats that have all their bits); the bounds are those of ordinary queries."""
    scale = 2.0 ** max(-power, -120) * D ** -0.5 if power > 0 else 2.0 ** min(-power, 120) * D ** -0.5
    c = Case([300, 40, 1, 0], H, hkv, D, 16, q_scale=2.0 ** power)
    c.check(*tt.attention_decode_q8(**c.args(), scale=scale), scale)


@pytest.mark.parametrize("power,scale", [(-100, 2.0 ** -60), (-110, 2.0 ** -30), (-126, 2.0 ** -100), (0, 2.0 ** -140)])
def test_scores_that_vanish(tt, power, scale):
    """q and scale both small: all keys count alike, and the places behind the last one do not."""
    c = Case([300, 41, 7, 0], 4, 2, 64, 16, q_scale=2.0 ** power)
    c.check(*tt.attention_decode_q8(**c.args(), scale=scale), scale)


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
    k[:, 0, 5] = 2.0 ** (rng.permutation(n) - 19)   # up to 2^3
    slots = c.table[0, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
    c.pools[0].write(slots, k)
    q = torch.zeros(2, G, 1, D)
    q[0, :, 0, 5] = 2.0 ** power * (1 + torch.arange(G) / 16)
    c.q = q.bfloat16()
    out, lse = tt.attention_decode_q8(**c.args())
    if power == 0:   # the others count, too
        c.check(out, lse)
        return
    kept, values, _ = c.rows(0)
    best = int(kept[:, 0, 5].argmax())
    want = c.q[0, :, 0, 5].double().numpy() * kept[best, 0, 5] * D ** -0.5
    assert (np.abs(lse[0, :, 0].double().cpu().numpy() - want) <= 2.0 ** -21 * want).all()
    assert np.array_equal(out[0, :, 0].double().cpu().numpy(), np.broadcast_to(values[best, 0], (G, D)))


@pytest.mark.parametrize("power", [18, 20, 22, 24, 26, 30, 60, 115])
@pytest.mark.parametrize("G,D,n", [(4, 128, 2000), (12, 64, 700), (2, 64, 90)])
def test_scores_beyond_the_exponents_range(tt, power, G, D, n):
    """Random keys and queries of 2^power: scores whose own last bit is more than one.  The largest is ahead of the others by more than a score and its value's
    exponent beside it may be off -- (D + 6) 2^-23 of sum |q k| and 2^-22 of the score -- so the result is its key's values (four bits each, a weight's 2^-11 does not
    reach bf16's last)."""
    c = Case([n], G, 1, D, 16, seed=G, q_scale=2.0 ** power)
    k, v, _ = (x[:, 0] for x in c.rows(0))
    q = c.q[0, :, 0].double().numpy()
    s = q @ k.T * D ** -0.5
    off = ((D + 6) * 2.0 ** -23 * D ** -0.5) * (np.abs(q) @ np.abs(k).T).max(-1) + 2.0 ** -22 * np.abs(s).max(-1)
    two = np.sort(s, -1)[:, -2:]
    sure = two[:, 1] - two[:, 0] > 2 * off + 60   # (60: nothing left of the second in the sum)
    out, lse = tt.attention_decode_q8(**c.args())
    assert sure.any()
    want = v[s.argmax(-1)]
    assert np.array_equal(out[0, :, 0].double().cpu().numpy()[sure], want[sure])
    assert (np.abs(lse[0, :, 0].double().cpu().numpy() - two[:, 1]) <= off + 2.0 ** -20 * np.abs(two[:, 1]))[sure].all()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def whole_scores(G, D, n, q, one, other, at):
    """A sequence of n keys whose scores in base 2 are whole numbers, taken without rounding: q one = q's channels times those of a key, `other` those of the key `at`.
    Values' exponents are 0.  -> the case, and the scale whose product with log2 e is 1 in 32 bits."""
    scale = np.float32(0.69314718)
    while scale * np.float32(1.4426950408889634) < 1:
        scale = np.nextafter(scale, np.float32(1))
    assert scale * np.float32(1.4426950408889634) == 1
    c = Case([n], G, 1, D, 16)
    k = np.zeros((n, 1, D))
    k[:, 0, :2] = one
    k[at, 0, :2] = other
    slots = c.table[0, np.arange(n) // 16].astype(np.int64) * 16 + np.arange(n) % 16
    c.pools[0].write(slots, k)
    v = np.random.default_rng(n).uniform(-448, 448, (n, 1, D))
    v[:, 0, 2] = 448
    c.pools[1].write(slots, v)
    c.q = torch.zeros(1, G, 1, D)
    c.q[..., :2] = torch.tensor(q)
    c.q = c.q.bfloat16()
    kept, _, ev = c.rows(0)
    assert np.array_equal(kept, k) and not ev.any()
    return c, float(scale)


FAR = [  # q's channels, those of all keys but one, that one's, and how much its score (base 2) is ahead: a few of the scores' last bits, or around 5, which raises the reference
    ((2.0 ** 24, 2.0), (1, 1), (1, 4), 6), ((2.0 ** 26, 8.0), (1, 0), (1, 1), 8), ((-2.0 ** 26, 8.0), (1, -1), (1, 0), 8), ((-2.0 ** 27, 16.0), (1, -1), (1, 0), 16),
    ((2.0 ** 10, 1.0), (1, 0), (1, 5), 5), ((2.0 ** 10, 1.0), (1, 0), (1, 6), 6), ((2.0 ** 20, 1.0), (1, 1), (1, 6), 5), ((2.0 ** 30, 128.0), (1, 0), (1, 1), 128)]


@pytest.mark.parametrize("q,one,other,ahead", FAR)
@pytest.mark.parametrize("G,D,n,at", [(1, 64, 50, 40), (8, 128, 50, 40), (16, 128, 100, 99), (12, 64, 180, 64), (2, 128, 40, 5)])
def test_a_key_a_little_above_far_scores(tt, q, one, other, ahead, G, D, n, at):
    """Scores and their differences are exact, so weights are powers of two: what is off is the exponential's 2^-22, the sums' (n / 16 + 40) 2^-23 and
    bf16's rounding.  The log-sum-exp is off by its constants' and its own roundings, 2^-21 of itself."""
    c, scale = whole_scores(G, D, n, q, one, other, at)
    out, lse = tt.attention_decode_q8(**c.args(), scale=scale)
    _, v, _ = c.rows(0)
    p = np.ones(n) * 2.0 ** -ahead
    p[at] = 1.0
    p /= p.sum()
    want = p @ v[:, 0]
    got = out[0, :, 0].double().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -21 + (n / 16 + 40) * 2.0 ** -23) * (p @ np.abs(v[:, 0]))).all()
    top = (q[0] * other[0] + q[1] * other[1]) * scale - np.log(p[at])
    assert (np.abs(lse[0, :, 0].double().cpu().numpy() - top) <= 2.0 ** -21 * abs(top) + 1e-6).all()


@pytest.mark.parametrize("q,one,other,ahead", FAR)
@pytest.mark.parametrize("G", [1, 16])
def test_far_scores_in_many_parts(tt, q, one, other, ahead, G):
    """Many sequences of the same pages, whose keys many warps share out.  What warps leave is merged by 32-bit log-sum-exps, which here tell scores apart no better than by their
    last bit, so a result is a mean of the values with weights that may be off by as much; finite it is."""
    c, scale = whole_scores(G, 64, 200, q, one, other, 60)
    a = c.args()
    a["q"] = a["q"].expand(1200, G, 1, 64).contiguous()
    a["block_table"], a["seq_lens"] = a["block_table"].expand(1200, -1).contiguous(), a["seq_lens"].expand(1200).contiguous()
    out, lse = tt.attention_decode_q8(**a, scale=scale)
    _, v, _ = c.rows(0)
    top = (q[0] * other[0] + q[1] * other[1]) * scale
    assert torch.isfinite(out).all() and (out.abs() <= 448).all()
    assert (out.double().cpu().numpy().min((0, 1, 2)) >= v[:, 0].min(0) - 2).all() and (out.double().cpu().numpy().max((0, 1, 2)) <= v[:, 0].max(0) + 2).all()
    assert (np.abs(lse.double().cpu().numpy() - top) <= 2.0 ** -20 * abs(top) + 6).all()


@pytest.mark.parametrize("power", [60, 100, 104, 110, 120, 127])
@pytest.mark.parametrize("G,D,n", [(1, 64, 50), (8, 128, 700), (16, 128, 100)])
def test_a_large_query_beside_blocks_of_large_keys(tt, power, G, D, n):
    """The head's largest value meets zeros only, and some blocks' scale is 2^40 for other channels' sake: scores are 0, though the query's scale times the
    block's is beyond 32 bits."""
    c = Case([n, 30], G, 1, D, 16)
    codes, powers = c.pools[0].parts()
    codes[..., 0] = 0
    powers[::2] = 104
    c.q = torch.zeros(2, G, 1, D)
    c.q[..., 0] = 2.0 ** power
    c.q = c.q.bfloat16()
    c.check(*tt.attention_decode_q8(**c.args()))
    # and one key that another channel, 2^25 below, meets: with the smallest code of a block of 2^40
    if power == 110:
        at = 20
        c.q[0, :, 0, 1] = 2.0 ** (power - 25)
        codes[..., 1] = 0
        codes[c.table[0, at // 16], 0, at % 16, 1] = 1
        powers[c.table[0, at // 16]] = 104
        out, lse = tt.attention_decode_q8(**c.args())
        k, v, _ = c.rows(0)
        top = 2.0 ** (power - 25) * k[at, 0, 1] * D ** -0.5
        assert top == 2.0 ** 116 * D ** -0.5
        assert np.array_equal(out[0, :, 0].double().cpu().numpy(), np.broadcast_to(v[at, 0], (G, D)))
        assert (np.abs(lse[0, :, 0].double().cpu().numpy() - top) <= 2.0 ** -21 * top).all()
