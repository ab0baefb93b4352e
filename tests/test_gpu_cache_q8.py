"""The 8-bit cache: bytes written equal to the format's definition, rows read back equal to the bit, everything else left alone."""
import numpy as np
import pytest

import q8_oracle as q8

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def as64(x):
    return x.double().cpu().numpy()


def same(got, want):
    """Bytes equal, but for the sign of NaN."""
    d = got != want
    return bool(((got[d] & 127) == 127).all() and ((want[d] & 127) == 127).all())


class Cache:
    def __init__(self, pages, hkv, page, D, fill=0x33):
        self.pools = [q8.Pool(pages, hkv, page, D, fill) for _ in range(2)]
        self.kc, self.vc = (dev(p.bytes) for p in self.pools)

    def append(self, tt, k, v, slots):
        slots = np.asarray(slots, np.int32)
        assert tt.cache_append_q8(k, v, dev(slots), self.kc, self.vc) == (self.kc, self.vc)
        for p, x, got in zip(self.pools, (k, v), (self.kc, self.vc)):
            p.write(slots, as64(x))
            assert same(got.cpu().numpy(), p.bytes)


def spread(T, hkv, D, dtype, seed=0):
    """Values whose size changes from token to token."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(T, hkv, D, generator=g, device="cuda") * (2 * torch.randn(T, hkv, 1, generator=g, device="cuda")).exp()).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hkv,D,page,pages", [(1, 1, 64, 16, 1), (1, 8, 128, 64, 3), (16, 1, 128, 16, 2), (45, 3, 64, 48, 2), (200, 8, 128, 32, 9), (513, 2, 64, 16, 40), (1000, 5, 128, 1024, 1),
                                                (31, 1, 128, 16, 3), (5000, 1, 64, 528, 10)])
def test_append_a_sequence(tt, T, hkv, D, page, pages, dtype):
    """Whole sequences at once, and then token by token and in small chunks, over pages in any order."""
    rng = np.random.default_rng(T)
    k, v = spread(T, hkv, D, dtype, 1), spread(T, hkv, D, dtype, 2)
    order = rng.permutation(pages)
    at = np.arange(T)
    slots = order[at // page] * page + at % page
    Cache(pages, hkv, page, D).append(tt, k, v, slots)
    c, t = Cache(pages, hkv, page, D), 0
    while t < T and t < 300:
        n = int(rng.choice([1, 1, 1, 2, 5, 20, 40]))
        c.append(tt, k[t:t + n], v[t:t + n], slots[t:t + n])
        t += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_batch_token_by_token(tt, dtype):
    B, hkv, D, page = 37, 4, 128, 32
    c = Cache(B * 2, hkv, page, D)
    lens = np.random.default_rng(1).integers(0, 30, B)
    for b in range(B):
        if lens[b]:
            at = np.arange(lens[b])
            c.append(tt, spread(lens[b], hkv, D, dtype, b), spread(lens[b], hkv, D, dtype, b + 50), (2 * b + at // page) * page + at % page)
    for step in range(20):
        at = lens + step
        c.append(tt, spread(B, hkv, D, dtype, 100 + step), spread(B, hkv, D, dtype, 200 + step), (2 * np.arange(B) + at // page) * page + at % page)


def test_growing_and_shrinking_tokens(tt):
    """Each token of a block larger than the ones before (its scale is raised fifteen times, twice too far for what it held), and each smaller."""
    hkv, D = 2, 64
    for sizes in (2.0 ** np.arange(0, 48, 3), 2.0 ** -np.arange(0, 48, 3), 2.0 ** np.arange(-60, 60, 8), [1, 1e30, 1e-30] * 5, [0.0] * 5 + [1.0] + [0.0] * 5):
        c = Cache(1, hkv, 16, D)
        for r, s in enumerate(sizes[:16]):
            x = spread(1, hkv, D, torch.float32, r)
            x = x / x.abs().amax() * float(s)
            c.append(tt, x, -2 * x, [r])


def test_a_block_begins_anew(tt):
    """A page given to another sequence: what its blocks held is forgotten with their first row, whatever bytes are there."""
    rng = np.random.default_rng(2)
    for T in (1, 7, 16, 20):
        c = Cache(2, 3, 32, 128)
        for p in c.pools:
            p.bytes[:] = rng.integers(0, 256, p.bytes.shape)
        c.kc, c.vc = (dev(p.bytes) for p in c.pools)
        c.append(tt, spread(T, 3, 128, torch.bfloat16, T) * 1e-3, spread(T, 3, 128, torch.bfloat16, T + 1) * 1e3, 32 + np.arange(T))
        # and a row of a block that is not its first, whose exponent is any byte
        c.append(tt, spread(1, 3, 128, torch.bfloat16, 5), spread(1, 3, 128, torch.bfloat16, 6), [5])


def test_rows_of_a_block_in_any_order(tt):
    c = Cache(3, 2, 48, 64)
    rng = np.random.default_rng(4)
    slots = np.concatenate([b * 16 + rng.permutation(16)[:n] for b, n in ((4, 16), (0, 3), (8, 9), (2, 1), (1, 12))])
    for seed in range(3):
        c.append(tt, spread(len(slots), 2, 64, torch.float32, seed), spread(len(slots), 2, 64, torch.float32, seed + 9), slots)


def test_slots_outside_and_empty(tt):
    k = torch.randn(9, 2, 64, device="cuda").bfloat16()
    c = Cache(2, 2, 16, 64)
    c.append(tt, k, -k, [-1, 3, 32, 31, -2 ** 31, 2 ** 31 - 1, 33, -5, -1])
    c.append(tt, k, -k, [-1] * 9)
    c.append(tt, k, -k, [-1, 4, -1, 20, 21, -1, 32, -1, -7])
    c.append(tt, k[:0], k[:0], [])
    Cache(0, 2, 16, 64).append(tt, k, k, range(9))


def test_one_slot_twice_stays_in_its_block(tt):
    """Not allowed, and what the block then holds is of any of the tokens; nothing else changes."""
    c = Cache(4, 2, 32, 128, fill=0)
    k = torch.randn(200, 2, 128, device="cuda")
    slots = torch.full((200,), 37, dtype=torch.int32, device="cuda")
    slots[100:] = torch.tensor([33, 70], device="cuda").repeat(50)
    slots[101::2] = 37
    before = c.kc.clone()
    tt.cache_append_q8(k, k, slots, c.kc, c.vc)
    at = 32 * 128
    before[1, :, :16 * 128], before[1, :, at] = c.kc[1, :, :16 * 128], c.kc[1, :, at]
    assert torch.equal(before, c.kc)


@pytest.mark.parametrize("D", [64, 128])
def test_strides_and_alignment(tt, D):
    T, H, hkv = 37, 4, 2
    rows = torch.randn(T, H + 2 * hkv, D, device="cuda").bfloat16()
    run = lambda k, v: Cache(3, hkv, 16, D).append(tt, k, v, range(T))
    run(rows[:, H:H + hkv], rows[:, H + hkv:])
    off = torch.randn(T * hkv * D + 1, device="cuda").bfloat16()[1:].view(T, hkv, D)
    run(off, rows[:, :hkv])
    odd = torch.randn(T, hkv, D + 1, device="cuda")[..., :D]
    run(odd, odd)
    heads = torch.randn(hkv, T, D, device="cuda").transpose(0, 1)
    run(heads, heads)
    one = torch.randn(1, hkv, D, device="cuda").expand(T, hkv, D)
    run(one, one)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_at_the_format_s_edges(tt, dtype):
    """Blocks whose largest value is at, just below and just above every exponent's reach, with values at and next to every border between two codes; and
    values that no exponent holds, infinities and NaN among others."""
    rng = np.random.default_rng(0)
    borders = (q8.POSITIVE[1:] + q8.POSITIVE[:-1]) / 2
    rows = []
    for e in range(q8.LOW - 1, q8.HIGH + 2):
        for top in (448.0, np.nextafter(np.float32(448), np.float32(0)), np.nextafter(np.float32(448), np.float32(np.inf))):
            block = np.zeros((16, 64))
            block[0, 0] = top
            block[1:3] = borders.reshape(2, 63)[:, :1].repeat(64, 1)
            block[1:3, :63] = borders.reshape(2, 63)
            block[3:5, :63] = np.nextafter(borders.astype(np.float32), np.float32(0)).reshape(2, 63)
            block[5:7, :63] = np.nextafter(borders.astype(np.float32), np.float32(np.inf)).reshape(2, 63)
            rows.append(block * 2.0 ** e * rng.choice([-1, 1], block.shape))
    for special in (0.0, -0.0, 1e-45, 1e-38, 1e-12, 448 * 2.0 ** 40, 449 * 2.0 ** 40, 3e38, np.inf, -np.inf, np.nan):
        block = rng.standard_normal((16, 64))
        block[5, 7] = special
        rows.append(block)
        rows.append(np.full((16, 64), special))
        rows.append(np.where(np.arange(64) % 2, special, rng.standard_normal((16, 64))))
    x = torch.from_numpy(np.concatenate(rows).astype(np.float32)).cuda().to(dtype).view(-1, 1, 64)
    T = x.shape[0]
    c = Cache(T // 16, 1, 16, 64)
    c.append(tt, x, -x.flip(0), range(T))
    # and onto what is there, each block's last row first
    c.append(tt, x.flip(0)[15::16], x[15::16], range(15, T, 16))


@pytest.mark.parametrize("hkv,D,page,lens", [(1, 64, 16, [1]), (8, 128, 64, [5, 0, 64, 130, 1]), (3, 64, 48, [0, 0, 7, 96, 0]), (2, 128, 16, [1000, 33]), (16, 64, 32, list(range(40))), (200, 128, 16, [3, 40]),
                                             (2, 64, 528, [529, 1100])])
def test_read(tt, hkv, D, page, lens):
    rng = np.random.default_rng(page)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + 3
    pool = [q8.Pool(pages, hkv, page, D) for _ in range(2)]
    for p in pool:
        p.bytes[:] = rng.integers(0, 256, p.bytes.shape)
        codes, powers = p.parts()
        codes[(codes & 127) == 127] = 0
    order = rng.permutation(pages)
    table = np.full((len(lens), max(per) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    total = int(cu[-1])
    want = [np.concatenate([p.rows(table[b], n) for b, n in enumerate(lens)]) for p in pool]
    kc, vc = (dev(p.bytes) for p in pool)
    for extra in (0, 21):
        k, v = (torch.full((total + extra, hkv, D), 3.0, device="cuda").bfloat16() for _ in range(2))
        got = tt.cache_read_q8(kc, vc, dev(table), dev(cu), total + extra, page, k=k, v=v)
        assert got[0] is k and got[1] is v
        for x, w in zip(got, want):
            assert np.array_equal(as64(x[:total]), w) and (x[total:] == 3.0).all()
    made = tt.cache_read_q8(kc, vc, dev(table), dev(cu), total, page)
    assert torch.equal(made[0], k[:total]) and torch.equal(made[1], v[:total])
    few = tt.cache_read_q8(kc, vc, dev(table), dev(cu), max(total - 5, 0), page)   # fewer rows asked for than there are
    assert torch.equal(few[0], k[:max(total - 5, 0)])
    off = torch.zeros(total * hkv * D + 8, device="cuda").bfloat16()[8:].view(total, hkv, D)   # rows on 16 bytes, not on 32
    assert torch.equal(tt.cache_read_q8(kc, vc, dev(table), dev(cu), total, page, k=off)[0], k[:total])


def test_read_of_pages_outside_and_nan(tt):
    kc, vc = tt.cache_alloc_q8(3, 2, 16, 64)
    x = torch.randn(48, 2, 64, device="cuda")
    tt.cache_append_q8(x, x, torch.arange(48, dtype=torch.int32, device="cuda"), kc, vc)
    kc[1, 0, 5 * 64 + 3] = 0x7f
    kc[1, 0, 5 * 64 + 4] = 0xff
    table = torch.tensor([[1, -1, 0], [3, 2, 2 ** 30]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 48, 100], dtype=torch.int32, device="cuda")
    k, v = tt.cache_read_q8(kc, vc, table, cu, 100, 16)
    assert not v[16:32].any() and not v[48:64].any() and not v[80:96].any() and not k[96:].any()   # (the last four lie behind the table's width)
    assert torch.isnan(k[5, 0, 3:5]).all() and int(torch.isnan(k).sum()) == 2 and torch.equal(v[32:48], tt.cache_read_q8(kc, vc, table[:, 2:].contiguous(), torch.tensor([0, 16, 16], dtype=torch.int32, device="cuda"), 16, 16)[1])


def test_streams_and_graphs(tt):
    c, d = Cache(8, 2, 32, 128), Cache(8, 2, 32, 128)
    slots = torch.arange(200, dtype=torch.int32, device="cuda")
    k, v = spread(200, 2, 128, torch.bfloat16, 1), spread(200, 2, 128, torch.bfloat16, 2)
    tt.cache_append_q8(k, v, slots, c.kc, c.vc)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tt.cache_append_q8(k, v, slots, d.kc, d.vc)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c.kc, d.kc) and torch.equal(c.vc, d.vc)
    table, cu = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8), torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tt.cache_append_q8(k, v, slots, d.kc, d.vc)
        got = tt.cache_read_q8(d.kc, d.vc, table, cu, 200, 32)
    k.normal_(), v.normal_()
    graph.replay()
    tt.cache_append_q8(k, v, slots, c.kc, c.vc)
    assert torch.equal(c.kc, d.kc) and all(torch.equal(a, b) for a, b in zip(got, tt.cache_read_q8(c.kc, c.vc, table, cu, 200, 32)))


def test_refusals(tt):
    kc, vc = tt.cache_alloc_q8(4, 2, 16, 64)
    assert kc.shape == (4, 2, 16 * 64 + 32) and tt.cache_alloc_q8(1, 1, 528, 128)[0].shape[2] == 528 * 128 + 64
    k, slots = torch.randn(5, 2, 64, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")
    table, cu = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    for bad in (dict(page_size=24), dict(page_size=0), dict(head_dim=96)):
        with pytest.raises(ValueError):
            tt.cache_alloc_q8(**{**dict(pages=1, kv_heads=1, page_size=16, head_dim=64), **bad})
    q4 = tt.cache_alloc_q4(4, 2, 16, 64)
    for bad in (dict(k=k.half()), dict(k=k[:, :1]), dict(v=k[:4]), dict(k=k[..., :32]), dict(slots=slots.long()), dict(slots=slots[:4]), dict(k=k.cpu()), dict(k_cache=vc), dict(k_cache=kc[:3]),
                dict(k_cache=kc.view(torch.int8)), dict(k_cache=q4[0], v_cache=q4[1]), dict(k=kc.view(-1)[:2560].view(torch.float32).view(5, 2, 64)), dict(k=k.transpose(1, 2))):
        with pytest.raises((ValueError, RuntimeError)):
            tt.cache_append_q8(**{**dict(k=k, v=k + 1, slots=slots, k_cache=kc, v_cache=vc), **bad})
    for bad in (dict(block_table=table.long()), dict(cu_lens=cu.long()), dict(cu_lens=cu[:1]), dict(page_size=32), dict(page_size=17), dict(total=-1), dict(total=2 ** 40), dict(k=torch.zeros(20, 2, 64, device="cuda")),
                dict(k_cache=q4[0], v_cache=q4[1]), dict(block_table=table[0])):
        with pytest.raises(ValueError):
            tt.cache_read_q8(**{**dict(k_cache=kc, v_cache=vc, block_table=table, cu_lens=cu, total=20, page_size=16), **bad})
