"""Decode over the 4-bit cache against attention in 64 bits over what the cache holds.

Bound per output value.  Unpacked keys and values and the shifted q are exact, a product of two is exact in 32 bits, so with
u = 2^-23 (a truncated addition) a score is off by at most ds = scale (D + 2) u sum |q k|.  A probability is then off by ds, by the
exponential's 2^-22 and by half a step of half precision, 2^-11 (or 2^-35 of the row's largest, all together n 2^-35).  The sums over the
n keys, in steps of 16, are off by (n / 16 + 40) u of sum p |v|, and bf16 rounds the result by 2^-8 of it.  The log-sum-exp is off by ds, the
exponentials and its own sum, and by 2^-22 of itself."""
import math

import numpy as np
import pytest

import q4_oracle as q4

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -23


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def sequence(q, k, v, scale):
    """q [G, D], k, v [n, D] -> (out, lse, bound of out, bound of lse)."""
    n, D = k.shape
    if n == 0:
        return np.zeros_like(q), np.full(len(q), -np.inf), np.zeros_like(q), np.zeros(len(q))
    s = q @ k.T * scale
    ds = (D + 2) * U * scale * (np.abs(q) @ np.abs(k).T).max(-1)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - top)
    den = p.sum(-1, keepdims=True)
    out, lse = p @ v / den, (top + np.log(den))[:, 0]
    weight = p @ np.abs(v) / den
    rel = 2 * np.expm1(ds) + 2.0 ** -21 + 2.0 ** -11 + n * 2.0 ** -35 + (n / 16 + 40) * U
    # (1.0625: to the fourth, for products of the relative errors; and the subnormal probabilities of every value)
    bound = 1.0625 * (rel[:, None] * weight + n * 2.0 ** -35 * np.abs(v).max(0)) + 2.0 ** -8 * np.abs(out)
    return out, lse, bound, 1.0625 * (ds + 2.0 ** -21 + (n / 16 + 40) * U + 2.0 ** -22 * np.abs(lse)) + 1e-6


class Case:
    def __init__(self, lens, H, hkv, D, page, seed=0, table=True, spare=3, sigma=1.0, q_scale=1.0, fill=0xFF, width=0, q=None):
        rng = np.random.default_rng(seed)
        self.lens, self.H, self.hkv, self.D, self.page = lens, H, hkv, D, page
        B = len(lens)
        per = [-(-n // page) for n in lens] if table else [1] * B
        self.pages = sum(per) + (spare if table else 0)
        order = rng.permutation(self.pages) if table else np.arange(B)
        self.table = np.full((B, max(max(per), 1) + width), -1, np.int32)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n]
            at += n
        # rows that no sequence owns hold NaN scales
        self.pools = [q4.Pool(self.pages, hkv, page, D, fill) for _ in range(2)]
        for b, n in enumerate(lens):
            at = np.arange(n)
            slots = self.table[b, at // page].astype(np.int64) * page + at % page
            for pool in self.pools:
                pool.write(slots, rng.standard_normal((n, hkv, D)).astype(np.float32) * sigma)
        self.use_table = table
        self.q = (rng.standard_normal((B, H, 1, D)) * q_scale if q is None else q).astype(np.float32)
        self.q = torch.from_numpy(self.q).bfloat16()

    def args(self):
        return dict(q=self.q.cuda(), k_cache=dev(self.pools[0].bytes), v_cache=dev(self.pools[1].bytes), block_table=dev(self.table) if self.use_table else None,
                    seq_lens=dev(np.array(self.lens, np.int32)))

    def rows(self, b, n=None):
        return (p.rows(self.table[b], self.lens[b] if n is None else n) for p in self.pools)

    def check(self, out, lse, scale=None):
        scale = self.D ** -0.5 if scale is None else scale
        q, G = self.q.double().numpy(), self.H // self.hkv
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        for b in range(len(self.lens)):
            k, v = self.rows(b)
            for h in range(self.hkv):
                at = slice(h * G, (h + 1) * G)
                o, y, bo, by = sequence(q[b, at, 0], k[:, h], v[:, h], scale)
                assert (np.abs(out[b, at, 0] - o) <= bo).all(), (b, h, float((np.abs(out[b, at, 0] - o) / np.maximum(bo, 1e-30)).max()))
                if self.lens[b] == 0:
                    assert (lse[b, at, 0] == -np.inf).all()
                else:
                    assert (np.abs(lse[b, at, 0] - y) <= by).all(), (b, h, float((np.abs(lse[b, at, 0] - y) / by).max()))


@pytest.mark.parametrize("lens,H,hkv,D,page", [
    ([1], 1, 1, 64, 16), ([1], 8, 8, 128, 64), ([1, 2, 15, 16, 17], 4, 2, 128, 16), ([0, 31, 32, 33, 0, 127, 128, 129], 6, 2, 64, 16), ([255, 256, 257, 511, 513], 8, 1, 128, 32),
    ([100, 700], 7, 1, 128, 48), ([333, 5], 9, 1, 128, 64), ([300, 1, 0], 12, 1, 64, 48), ([500, 64], 16, 1, 128, 128), ([400], 17, 1, 128, 16), ([260, 3], 40, 2, 64, 64),
    ([129], 33, 1, 128, 256), ([0, 31, 32, 33, 0, 127, 128, 5], 40, 2, 64, 16), ([128, 0, 100], 24, 1, 128, 64), ([0, 0], 3, 1, 128, 16), (list(range(97)), 6, 2, 64, 16), ([5001], 32, 8, 128, 64), ([3000, 1, 2999], 5, 1, 64, 80), ([4097], 2, 2, 128, 1024)])
def test_against_64_bits(tt, lens, H, hkv, D, page):
    c = Case(lens, H, hkv, D, page, seed=len(lens) + H)
    a = c.args()
    out, lse = tt.attention_decode_q4(**a)
    c.check(out, lse)
    # a shorter bound on the lengths divides the keys in another way
    c.check(*tt.attention_decode_q4(**a, max_len=max(max(lens), 1)))
    out2, lse2 = tt.attention_decode_q4(**a, scale=0.3)
    c.check(out2, lse2, 0.3)


@pytest.mark.parametrize("B,H,hkv,D,page", [(3, 8, 2, 128, 64), (2, 4, 4, 64, 512)])
def test_without_a_block_table(tt, B, H, hkv, D, page):
    c = Case([page] * B, H, hkv, D, page, table=False)
    a = c.args()
    a["seq_lens"] = None
    c.check(*tt.attention_decode_q4(**a))
    c = Case([page, 1, 0][:B], H, hkv, D, page, table=False)
    c.check(*tt.attention_decode_q4(**c.args()))


def test_many_slices_and_one_long_sequence(tt):
    for lens, H, hkv in (([200 + 7 * i for i in range(40)], 16, 16), ([40000], 2, 1), ([20000, 9], 16, 1)):
        c = Case(lens, H, hkv, 64, 64)
        c.check(*tt.attention_decode_q4(**c.args()))


@pytest.mark.parametrize("B,H,hkv,D,longest", [(16, 32, 4, 128, 900), (10, 128, 8, 128, 700), (12, 64, 4, 64, 900), (20, 64, 4, 64, 700), (3, 300, 1, 64, 2500), (700, 2, 1, 64, 70)])
def test_many_rows_of_many_parts(tt, B, H, hkv, D, longest):
    """Every width of the merge, with a short and an empty sequence among the others; and nothing but empty ones."""
    rng = np.random.default_rng(B)
    lens = rng.integers(longest // 2, longest + 1, B).tolist()
    lens[B // 2], lens[-1] = 0, 1
    c = Case(lens, H, hkv, D, 16)
    a = c.args()
    c.check(*tt.attention_decode_q4(**a))
    a["seq_lens"].zero_()
    out, lse = tt.attention_decode_q4(**a)
    assert not out.any() and (lse == -np.inf).all()


@pytest.mark.parametrize("G", [1, 8, 16])
def test_scores_that_rise(tt, G):
    """Every tile's scores pass the ones before: the reference is raised again and again, in every warp and range."""
    D, page, n = 128, 16, 1500
    c = Case([n], G, 1, D, page)
    ramp = np.zeros((n, 1, D))
    ramp[:, 0, 0] = np.linspace(-200, 200, n)
    slots = c.table[0, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
    c.pools[0].write(slots, ramp)
    c.q = torch.zeros(1, G, 1, D)
    c.q[..., 0] = torch.linspace(-4, 4, G + 1)[1:].view(1, G, 1)
    c.q = c.q.bfloat16()
    c.check(*tt.attention_decode_q4(**c.args()))


def test_one_key_takes_nearly_all(tt):
    """A sink: its probability is 2^20 times the others', which are in the subnormal range of half together."""
    D, page, n = 64, 64, 3000
    c = Case([n], 4, 1, D, page, sigma=0.01)
    k = np.zeros((1, 1, D))
    k[0, 0, :32] = 1.0
    c.pools[0].write(c.table[0, :1].astype(np.int64) * page, k)
    c.q = torch.full((1, 4, 1, D), 0.0)
    c.q[..., :32] = 14.0 * 8 / 32
    c.q = c.q.bfloat16()
    c.check(*tt.attention_decode_q4(**c.args()))


@pytest.mark.parametrize("q_scale", [0.0, 1e-37, 1e-20, 1e-3, 1e4])
def test_sizes_of_q(tt, q_scale):
    c = Case([300, 40], 4, 2, 128, 16, q_scale=q_scale, sigma=1.0 if q_scale <= 1 else 1e-4)
    c.check(*tt.attention_decode_q4(**c.args()))


def test_one_value_of_q_above_the_others(tt):
    """q in half keeps the small values beside a large one: 2^-20 of it."""
    c = Case([300], 2, 1, 64, 16)
    q = c.q.float()
    q[..., 0] = 2.0 ** 12
    q[..., 1:] = q[..., 1:].sign() * 2.0 ** -8
    c.q = q.bfloat16()
    rows = c.pools[0]
    nib = rows._parts()[0]
    nib[..., 0] = nib[..., 0] & 0xF0 | 8   # the first channel of every key is 0
    for b in range(1):
        c.check(*tt.attention_decode_q4(**c.args()))


def test_what_lies_behind_the_end_does_not_matter(tt):
    for lens in ([1, 17, 33, 500], [0, 15, 129, 130]):
        c = Case(lens, 8, 2, 128, 64)
        a = c.args()
        want = tt.attention_decode_q4(**a)
        assert all(torch.isfinite(w[torch.isfinite(w)]).all() and not torch.isnan(w).any() for w in want)
        for pool, name in zip(c.pools, ("k_cache", "v_cache")):
            data, codes = pool._parts()
            owned = np.zeros(codes.shape[:1] + codes.shape[2:3], bool)
            for b, n in enumerate(lens):
                at = np.arange(n)
                owned[c.table[b, at // 64], at % 64] = True
            free = ~owned[:, None, :, None] & np.ones_like(codes, bool)
            codes[free] = np.random.default_rng(1).integers(0, 256, int(free.sum()))
            a[name] = dev(pool.bytes)
        assert all(torch.equal(x, y) for x, y in zip(want, tt.attention_decode_q4(**a)))


def test_pages_outside_the_pool_have_no_keys(tt):
    c = Case([100, 70, 40], 4, 1, 64, 16, width=2)
    c.table[0, 2], c.table[0, 6], c.table[1, 0], c.table[2, :] = -1, c.pages, 2 ** 30, -2 ** 31
    out, lse = tt.attention_decode_q4(**c.args())
    q = c.q.double().numpy()
    for b, n in enumerate(c.lens):
        at = np.array([r for r in range(n) if 0 <= c.table[b, r // 16] < c.pages], int)
        full = c.table[b].copy()
        full[(full < 0) | (full >= c.pages)] = 0
        k, v = (p.rows(full, n)[at] for p in c.pools)
        o, y, bo, by = sequence(q[b, :, 0], k[:, 0], v[:, 0], 0.125)
        assert (np.abs(out[b, :, 0].double().cpu().numpy() - o) <= bo).all()
        got = lse[b, :, 0].double().cpu().numpy()
        assert (got == -np.inf).all() if len(at) == 0 else (np.abs(got - y) <= by).all()


def test_lengths_are_clamped(tt):
    c = Case([96, 96], 2, 1, 64, 16)
    a = c.args()
    want = tt.attention_decode_q4(**a)
    a["seq_lens"] = torch.tensor([2 ** 31 - 1, 97], dtype=torch.int32, device="cuda")
    assert all(torch.equal(x, y) for x, y in zip(want, tt.attention_decode_q4(**a)))
    a["seq_lens"] = torch.tensor([-5, -2 ** 31], dtype=torch.int32, device="cuda")
    out, lse = tt.attention_decode_q4(**a)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_nan_and_infinity(tt):
    c = Case([40, 40, 40, 40], 4, 1, 64, 16)
    q = c.q.float()
    q[1, 2, 0, 5], q[2, 1, 0, 7] = float("nan"), float("inf")
    c.q = q.bfloat16()
    data, codes = c.pools[1]._parts()
    codes[c.table[3, 1], 0, 3, 1] = 255     # a value's group of channels 32 .. 63
    out, lse = tt.attention_decode_q4(**c.args())
    bad = torch.isnan(out)[:, :, 0].cpu()
    assert bad[1, 2].all() and bad[2, 1].all() and bad[3, :, 32:].all()
    assert int(bad.sum()) == 64 + 64 + 4 * 32
    codes[c.table[3, 1], 0, 3, 1] = 10
    c.pools[0]._parts()[1][c.table[0, 0], 0, 2, 0] = 255   # a key's group: the whole row
    out, lse = tt.attention_decode_q4(**c.args())
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and not torch.isnan(out[3]).any()


def test_beyond_4_gb(tt):
    hkv, page, D = 8, 128, 128
    per = hkv * page * q4.row_bytes(D)
    pages = (1 << 32) // per + 40
    c = Case([300, 129], 8, hkv, D, page, spare=0)
    a = c.args()
    want = tt.attention_decode_q4(**a)
    pools = [torch.empty(pages, hkv, page * q4.row_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2)]
    far = torch.tensor([pages - 1 - i * 7 for i in range(c.pages)], device="cuda")
    for p, name in zip(pools, ("k_cache", "v_cache")):
        p[far] = a[name]
        a[name] = p
    t = a["block_table"].long()
    a["block_table"] = torch.where(t >= 0, far[t.clamp_min(0)], -1).int()
    assert all(torch.equal(x, y) for x, y in zip(want, tt.attention_decode_q4(**a)))
    # and rows written and read there
    x = torch.randn(40, hkv, D, device="cuda").bfloat16()
    slots = ((pages - 3) * page + torch.arange(40, device="cuda")).int()
    tt.cache_append_q4(x, x, slots, *pools)
    small = tt.cache_append_q4(x, x, torch.arange(40, dtype=torch.int32, device="cuda"), *tt.cache_alloc_q4(1, hkv, page, D))
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    got = tt.cache_read_q4(*pools, torch.tensor([[pages - 3]], dtype=torch.int32, device="cuda"), cu, 40, page)
    assert all(torch.equal(x, y) for x, y in zip(got, tt.cache_read_q4(*small, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), cu, 40, page)))


def test_repeats_streams_and_graphs(tt):
    c = Case([2000, 77, 0], 16, 2, 128, 64)
    a = c.args()
    want = tt.attention_decode_q4(**a)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(tt.attention_decode_q4(**a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r in got for x, y in zip(want, r))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = tt.attention_decode_q4(**a)
    other = Case([1500, 3, 60], 16, 2, 128, 64, seed=5)
    b = other.args()
    for name in ("q", "seq_lens"):
        a[name].copy_(b[name])
    a["block_table"].fill_(0)
    n = min(a["block_table"].shape[1], b["block_table"].shape[1])
    a["block_table"][:, :n] = b["block_table"][:, :n]
    m = min(a["k_cache"].shape[0], b["k_cache"].shape[0])
    for name in ("k_cache", "v_cache"):
        a[name].zero_()
        a[name][:m] = b[name][:m]
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((out, lse), tt.attention_decode_q4(**a)))
    assert m == b["k_cache"].shape[0]
    other.check(out, lse)


def test_outputs_given_and_neighbouring_memory(tt):
    from test_gpu_canary import Guarded
    for lens, H, hkv, D in (([1], 1, 1, 64), ([1300, 5], 6, 2, 128), ([700], 20, 1, 64)):
        c = Case(lens, H, hkv, D, 16)
        a = c.args()
        B = len(lens)
        d = tt.capi.make_desc(B, H, 1, c.table.shape[1] * 16, D, tt.capi.TT_BF16, False, None, Hkv=hkv)
        import ctypes
        need = int(tt.capi.lib.tt_attn_decode_q4_workspace_bytes(ctypes.byref(d)))
        out, lse, ws = Guarded((B, H, 1, D), torch.bfloat16), Guarded((B, H, 1), torch.float32), Guarded((max(need, 256),), torch.uint8)
        got = tt.attention_decode_q4(**a, out=out.t, lse=lse.t, workspace=ws.t)
        torch.cuda.synchronize()
        assert got[0] is out.t and got[1] is lse.t and out.intact() and lse.intact() and ws.intact()
        c.check(*got)
        o, none = tt.attention_decode_q4(**a, need_lse=False)
        assert none is None and torch.equal(o, out.t)


def test_refusals(tt):
    c = Case([50, 20], 4, 2, 64, 16)
    a = c.args()
    tt.attention_decode_q4(**a)
    q, t, n = a["q"], a["block_table"], a["seq_lens"]
    for kw in (dict(q=q.float()), dict(q=q[:, :, 0]), dict(q=q.expand(2, 4, 2, 64)), dict(q=q.cpu()), dict(q=q[:, :3].contiguous()), dict(q=torch.zeros(2, 4, 1, 128, device="cuda").bfloat16()),
               dict(q=torch.zeros(2, 4, 1, 32, device="cuda").bfloat16()), dict(k_cache=a["k_cache"].int()), dict(v_cache=a["v_cache"][:1]), dict(k_cache=a["k_cache"].cpu()),
               dict(block_table=t.long()), dict(block_table=t[:1]), dict(block_table=t[0]), dict(block_table=None), dict(seq_lens=n.long()), dict(seq_lens=n[:1]), dict(max_len=10 ** 6),
               dict(max_len=2 ** 32 + 16), dict(max_len=0), dict(out=torch.zeros(2, 4, 1, 64, device="cuda")), dict(out=q[:1]), dict(out=q), dict(lse=torch.zeros(2, 4, device="cuda")), dict(workspace=5),
               dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            tt.attention_decode_q4(**{**a, **kw})
    with pytest.raises(TypeError):
        tt.attention_decode_q4(**a, max_len=[1])
