"""Keys and values into a paged cache with rotation (and norm) on the way, against 64 bits; the bounds are those of norm_rotary_oracle, values that
are only copied are equal to the bit, and rows that no token goes to keep what they hold."""
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


class Case:
    def __init__(self, tt, T, H, Hkv, D, R, page, pages, dtype=torch.bfloat16, normed=True, seed=0, layout="fused"):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        rows = torch.randn(T, H + 2 * Hkv, D, generator=g, device="cuda").to(dtype)
        self.q, self.k, self.v = rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:]
        if layout == "apart":
            self.q, self.k, self.v = (x.contiguous() for x in (self.q, self.k, self.v))
        if layout == "odd":   # rows that start anywhere
            pad = torch.zeros(T, H + 2 * Hkv, D + 1, device="cuda", dtype=dtype)
            pad[..., 1:] = rows
            self.q, self.k, self.v = pad[:, :H, 1:], pad[:, H:H + Hkv, 1:], pad[:, H + Hkv:, 1:]
        self.pools = [torch.randn(pages, Hkv, page, D, generator=g, device="cuda").bfloat16() for _ in range(2)]
        self.page = page
        slots = self.rng.permutation(pages * page)[:T].astype(np.int32)
        self.slots = torch.from_numpy(slots).cuda()
        self.pos = torch.from_numpy(self.rng.integers(0, 100000, T).astype(np.int32)).cuda()
        self.freq, _ = tt.rotary_frequencies(R)
        self.w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype if seed % 2 else torch.float32) for _ in range(2)] if normed else [None, None]

    def call(self, tt, **kw):
        how = dict(q_weight=self.w[0] if kw.get("q", self.q) is not None else None, k_weight=self.w[1])
        a = {**dict(q=self.q, k=self.k, v=self.v, slots=self.slots, positions=self.pos, inv_freq=self.freq, k_pool=self.pools[0], v_pool=self.pools[1]), **how, **kw}
        return tt.cache_append_rotary(**a)

    def check(self, tt, interleaved=False, scale=None, with_q=True, with_k=False):
        before = [p.clone() for p in self.pools]
        t = nr.angles(self.pos.cpu().numpy()[None], self.freq.tolist(), None)[:, None]
        s = 1.0 if scale is None else scale
        w = [None if x is None else host(x) for x in self.w]
        also = torch.full(self.k.shape, 5.0, device="cuda", dtype=torch.bfloat16) if with_k else None
        got = self.call(tt, interleaved=interleaved, scale=scale, out_k=also, **({} if with_q else dict(q=None)))
        if with_q:
            assert got.dtype == torch.bfloat16 and got.is_contiguous()
            near(got, *nr.forward(host(self.q), w[0], t, interleaved, s))
        else:
            assert got is None
        slots = self.slots.cpu().numpy()
        kept = (slots >= 0) & (slots < self.pools[0].shape[0] * self.page)
        at = torch.from_numpy(slots[kept].astype(np.int64)).cuda()
        want, bound = nr.forward(host(self.k), w[1], t, interleaved, s)
        rows = self.pools[0][at // self.page, :, at % self.page]
        near(rows, want[kept], bound[kept])
        keep = torch.from_numpy(np.nonzero(kept)[0]).cuda()
        assert torch.equal(self.pools[1][at // self.page, :, at % self.page], self.v[keep].bfloat16())
        if with_k:
            assert torch.equal(also[keep], rows)
            near(also, want, bound)
        for p, b in zip(self.pools, before):
            b[at // self.page, :, at % self.page] = p[at // self.page, :, at % self.page]
            assert torch.equal(p, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,Hkv,D,R,page,pages,normed", [(1, 1, 1, 64, 64, 16, 1, False), (1, 32, 8, 128, 128, 64, 3, True), (64, 32, 8, 128, 64, 16, 9, True), (37, 6, 3, 64, 32, 1, 50, False),
                                                          (200, 4, 1, 128, 2, 7, 40, True), (2100, 4, 4, 64, 64, 128, 17, True), (513, 16, 1, 128, 128, 48, 11, False)])
def test_shapes(tt, T, H, Hkv, D, R, page, pages, normed, dtype):
    for i, layout in enumerate(("fused", "apart", "odd")):
        c = Case(tt, T, H, Hkv, D, R, page, pages, dtype, normed, seed=T + i, layout=layout)
        c.check(tt, interleaved=i == 1, scale=(None, 0.5, None)[i], with_q=i != 2, with_k=i != 0)


@pytest.mark.parametrize("normed", [False, True])
def test_slots_that_are_passed_over(tt, normed):
    c = Case(tt, 90, 4, 2, 128, 128, 16, 8, normed=normed)
    c.slots[::3] = -1
    c.slots[1::9] = 8 * 16
    c.slots[2] = 2 ** 31 - 1
    c.slots[4] = -2 ** 31
    c.check(tt, with_k=True)
    c.slots.fill_(-1)
    c.check(tt)
    no_pages = torch.empty(0, 2, 16, 128, device="cuda", dtype=torch.bfloat16)
    c.slots.fill_(0)
    before = c.pools[0].clone()
    c.call(tt, k_pool=no_pages, v_pool=no_pages)
    assert torch.equal(c.pools[0], before)


def test_in_place_and_no_tokens(tt):
    c = Case(tt, 33, 4, 2, 64, 32, 16, 5)
    want = c.call(tt)
    pools = [p.clone() for p in c.pools]
    k = c.pools[0][c.slots.long() // 16, :, c.slots.long() % 16]
    got = c.call(tt, out_q=c.q, out_k=c.k)
    assert got is c.q and torch.equal(c.q, want) and torch.equal(c.k, k) and all(torch.equal(a, b) for a, b in zip(pools, c.pools))
    empty = lambda x: x[:0]
    got = c.call(tt, q=empty(c.q), k=empty(c.k), v=empty(c.v), slots=c.slots[:0], positions=c.pos[:0])
    assert got.shape == (0, 4, 64)


def test_as_rotary_and_a_copy(tt):
    """Without weights the keys are those of `rotary_forward`, and with them those of `norm_rotary_forward`, to the bit."""
    for normed in (False, True):
        c = Case(tt, 77, 8, 2, 128, 128, 16, 6, normed=normed, seed=1)
        got = c.call(tt)
        q, k = tt.norm_rotary_forward(c.q, c.k, *c.w, c.pos, c.freq) if normed else tt.rotary_forward(c.q, c.k, c.pos, c.freq)
        at = c.slots.long()
        assert torch.equal(got, q) and torch.equal(c.pools[0][at // 16, :, at % 16], k)


def test_other_streams_and_graphs(tt):
    c = Case(tt, 64, 8, 2, 128, 128, 64, 4)
    want = c.call(tt)
    pools = [p.clone() for p in c.pools]
    side = torch.cuda.Stream()
    for p in c.pools:
        p.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.call(tt)
    torch.cuda.current_stream().wait_stream(side)
    at = c.slots.long()
    for p, b in zip(c.pools, pools):
        assert torch.equal(got, want) and torch.equal(p[at // 64, :, at % 64], b[at // 64, :, at % 64])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.call(tt)
    c.k.normal_(), c.q.normal_(), c.pos.add_(3)
    graph.replay()
    first = [p.clone() for p in c.pools]
    assert torch.equal(got, c.call(tt)) and all(torch.equal(a, b) for a, b in zip(first, c.pools)) and not torch.equal(first[0], pools[0])


def test_refusals(tt):
    c = Case(tt, 12, 4, 2, 64, 64, 16, 4)
    f = torch.float32
    for bad in (dict(v=c.v[:, :1]), dict(v=c.v.float()), dict(slots=c.slots.long()), dict(slots=c.slots[:5]), dict(slots=c.slots[::2]), dict(k_pool=c.pools[0].float()), dict(k_pool=c.pools[0][:, :1]),
                dict(v_pool=c.pools[1][:2]), dict(v_pool=c.pools[0]), dict(k_pool=c.pools[0].transpose(0, 2)), dict(positions=c.pos[:3]), dict(q_weight=None), dict(k_weight=None),
                dict(q=None, q_weight=c.w[0]), dict(q=None, q_weight=None, out_q=torch.empty(12, 4, 64, device="cuda", dtype=torch.bfloat16)), dict(q=c.q.float()), dict(out_q=torch.empty(12, 4, 64, device="cuda", dtype=f)),
                dict(out_k=torch.empty(12, 2, 64, device="cuda", dtype=f)), dict(out_k=c.pools[0].view(-1, 2, 64)[:12]), dict(eps=0.0), dict(k=None), dict(k=c.k.cpu()),
                dict(q=c.q[..., :32]), dict(out_q=c.k.new_empty(12, 4, 64).cpu())):
        with pytest.raises(ValueError):
            c.call(tt, **bad)
    x = Case(tt, 12, 4, 2, 32, 32, 16, 4)
    with pytest.raises((ValueError, tt.TTError)):
        x.call(tt)


def test_pools_beyond_4_gb(tt):
    """Rows whose places pass 32 bits, in elements and in bytes."""
    hkv, D, page = 8, 128, 64
    pages = (1 << 32) // (hkv * D * page) + 30
    pools = [torch.empty(pages, hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    T = 70
    rows = torch.randn(T, 4 + 2 * hkv, D, device="cuda").bfloat16()
    q, k, v = rows[:, :4], rows[:, 4:4 + hkv], rows[:, 4 + hkv:]
    slots = torch.cat((torch.arange(40), (pages - 1) * page + torch.arange(30))).int().cuda()
    freq, _ = tt.rotary_frequencies(D)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    got = tt.cache_append_rotary(q, k, v, slots, pos, freq, *pools)
    want_q, want_k = tt.rotary_forward(q, k, pos, freq)
    at = slots.long()
    assert torch.equal(got, want_q) and torch.equal(pools[0][at // page, :, at % page], want_k) and torch.equal(pools[1][at // page, :, at % page], v)
