"""The 4-bit cache: bytes written equal to the format's definition, rows read back equal to the bit, everything else left alone."""
import numpy as np
import pytest

import q4_oracle as q4

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def as64(x):
    return x.double().cpu().numpy()


def append_and_compare(tt, k, v, slots, pages, hkv, page, D, fill=0x5A):
    pools = [q4.Pool(pages, hkv, page, D, fill) for _ in range(2)]
    kc, vc = (dev(p.bytes) for p in pools)
    assert tt.cache_append_q4(k, v, dev(np.asarray(slots, np.int32)), kc, vc) == (kc, vc)
    for p, x, got in zip(pools, (k, v), (kc, vc)):
        p.write(slots, as64(x))
        assert np.array_equal(got.cpu().numpy(), p.bytes)
    return pools, kc, vc


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hkv,D,page,pages", [(1, 1, 64, 16, 1), (1, 8, 128, 64, 3), (16, 1, 128, 16, 2), (45, 3, 64, 48, 2), (200, 8, 128, 32, 9), (513, 2, 64, 16, 40), (1000, 5, 128, 128, 8)])
def test_append(tt, T, hkv, D, page, pages, dtype):
    rng = np.random.default_rng(T)
    k, v = (torch.randn(T, hkv, D, device="cuda").to(dtype) * s for s in (1.0, 30.0))
    append_and_compare(tt, k, v, rng.permutation(pages * page)[:T], pages, hkv, page, D)


def test_slots_outside_and_empty(tt):
    k = torch.randn(9, 2, 64, device="cuda").bfloat16()
    append_and_compare(tt, k, -k, [-1, 3, 32, 31, -2 ** 31, 2 ** 31 - 1, 0, 33, 16], 2, 2, 16, 64)
    append_and_compare(tt, k[:0], k[:0], [], 2, 2, 16, 64)
    append_and_compare(tt, k, k, range(9), 0, 2, 16, 64)


@pytest.mark.parametrize("D", [64, 128])
def test_strides_and_alignment(tt, D):
    T, H, hkv = 37, 4, 2
    rows = torch.randn(T, H + 2 * hkv, D, device="cuda").bfloat16()
    append_and_compare(tt, rows[:, H:H + hkv], rows[:, H + hkv:], range(T), 3, hkv, 16, D)
    off = torch.randn(T * hkv * D + 1, device="cuda").bfloat16()[1:].view(T, hkv, D)
    append_and_compare(tt, off, rows[:, :hkv], range(T), 3, hkv, 16, D)
    odd = torch.randn(T, hkv, D + 1, device="cuda")[..., :D]
    append_and_compare(tt, odd, odd, range(T), 3, hkv, 16, D)
    heads = torch.randn(hkv, T, D, device="cuda").transpose(0, 1)
    append_and_compare(tt, heads, heads, range(T), 3, hkv, 16, D)
    one = torch.randn(1, hkv, D, device="cuda").expand(T, hkv, D)
    append_and_compare(tt, one, one, range(T), 3, hkv, 16, D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_at_the_format_s_edges(tt, dtype):
    """Groups whose largest value is at, just below and just above every scale's reach, values at and next to every border between two
    levels, and values that no scale holds."""
    rng = np.random.default_rng(0)
    every = q4.scales(np.arange(q4.TOP + 1))
    rows = []
    for c in range(q4.TOP + 1):
        s = every[c]
        for top in (7.5 * s, np.nextafter(np.float32(7.5 * s), np.float32(0)), np.nextafter(np.float32(7.5 * s), np.float32(np.inf))):
            g = np.zeros(32)
            g[0] = top
            borders = (np.arange(-8, 8) + 0.5) * s
            g[1:17] = borders
            g[17:32] = np.nextafter(borders[:15].astype(np.float32), np.float32(rng.choice([-np.inf, np.inf])))
            rows.append(np.clip(g, -abs(top), abs(top)) if rng.random() < 0.5 else g)
    for special in (0.0, -0.0, 1e-45, 1e-38, 9e-7, 6720.0, 6721.0, 7000.0, 1e5, 3e38, np.inf, -np.inf, np.nan):
        g = rng.standard_normal(32)
        g[5] = special
        rows.append(g)
        rows.append(np.full(32, special))
        rows.append(np.where(np.arange(32) % 2, special, -special))
    for scale in 10.0 ** np.arange(-8, 6):
        rows.append(rng.standard_normal(32) * scale)
    n = len(rows) // 4 * 4
    x = torch.from_numpy(np.array(rows[:n] + rows[-4:], np.float32)).cuda().to(dtype).view(-1, 1, 128)
    T = x.shape[0]
    append_and_compare(tt, x, -x.flip(0), range(T), -(-T // 16), 1, 16, 128)


@pytest.mark.parametrize("hkv,D,page,lens", [(1, 64, 16, [1]), (8, 128, 64, [5, 0, 64, 130, 1]), (3, 64, 48, [0, 0, 7, 96, 0]), (2, 128, 16, [1000, 33]), (16, 64, 32, list(range(40))), (200, 128, 16, [3, 40])])
def test_read(tt, hkv, D, page, lens):
    rng = np.random.default_rng(page)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + 3
    pool = [q4.Pool(pages, hkv, page, D) for _ in range(2)]
    for p in pool:
        p.bytes[:] = rng.integers(0, 256, p.bytes.shape)
        p._parts()[1][:] = rng.integers(0, q4.TOP + 1, p._parts()[1].shape)   # (a view of the bytes)
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
        got = tt.cache_read_q4(kc, vc, dev(table), dev(cu), total + extra, page, k=k, v=v)
        assert got[0] is k and got[1] is v
        for x, w in zip(got, want):
            assert np.array_equal(as64(x[:total]), w) and (x[total:] == 3.0).all()
    made = tt.cache_read_q4(kc, vc, dev(table), dev(cu), total, page)
    assert torch.equal(made[0], k[:total]) and torch.equal(made[1], v[:total])
    # fewer rows asked for than there are
    few = tt.cache_read_q4(kc, vc, dev(table), dev(cu), max(total - 5, 0), page)
    assert torch.equal(few[0], k[:max(total - 5, 0)])


def test_read_without_a_page(tt):
    """Entries outside the pool, and tokens behind the table's width, give zeros."""
    kc, vc = tt.cache_alloc_q4(2, 1, 16, 64)
    x = torch.randn(32, 1, 64, device="cuda").bfloat16()
    tt.cache_append_q4(x, x, torch.arange(32, dtype=torch.int32, device="cuda"), kc, vc)
    table = torch.tensor([[1, -1, 0], [2, 1, 2 ** 30]], dtype=torch.int32, device="cuda")
    k, _ = tt.cache_read_q4(kc, vc, table, torch.tensor([0, 60, 108], dtype=torch.int32, device="cuda"), 108, 16)
    whole, _ = tt.cache_read_q4(kc, vc, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([0, 32], dtype=torch.int32, device="cuda"), 32, 16)
    assert torch.equal(k[:16], whole[16:]) and torch.equal(k[32:48], whole[:16]) and torch.equal(k[76:92], whole[16:])
    for a, b in ((16, 32), (48, 76), (92, 108)):
        assert (k[a:b] == 0).all()


def test_nan_stays_in_its_group(tt):
    kc, vc = tt.cache_alloc_q4(1, 1, 16, 128)
    x = torch.randn(3, 1, 128, device="cuda").bfloat16()
    x[1, 0, 40] = float("nan")
    tt.cache_append_q4(x, -x, torch.arange(3, dtype=torch.int32, device="cuda"), kc, vc)
    k, v = tt.cache_read_q4(kc, vc, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda"), 3, 16)
    for y in (k, v):
        bad = torch.isnan(y)
        assert bad[1, 0, 32:64].all() and int(bad.sum()) == 32


def test_an_error_is_at_most_half_a_step(tt):
    x = torch.randn(500, 4, 128, device="cuda") * torch.logspace(-4, 3, 500, device="cuda")[:, None, None]
    kc, vc = tt.cache_alloc_q4(32, 4, 16, 128)
    tt.cache_append_q4(x, x, torch.arange(500, dtype=torch.int32, device="cuda"), kc, vc)
    k, _ = tt.cache_read_q4(kc, vc, torch.arange(32, dtype=torch.int32, device="cuda")[None], torch.tensor([0, 500], dtype=torch.int32, device="cuda"), 500, 16)
    top = x.view(500, 4, 4, 32).abs().amax(-1, keepdim=True)
    # a scale is at most an eighth above what the largest value needs (its three bits of mantissa), and at least 2^-20
    half = (top / 7.5 * 1.125 / 2).clamp_min(2.0 ** -21) * (1 + 1e-6)
    assert ((k.float() - x).view(500, 4, 4, 32).abs() <= half).all()


def test_captured_append_and_read(tt):
    T, hkv, D, page = 50, 2, 128, 16
    kc, vc = tt.cache_alloc_q4(8, hkv, page, D)
    k, v = (torch.randn(T, hkv, D, device="cuda").bfloat16() for _ in range(2))
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    table, cu = torch.arange(8, dtype=torch.int32, device="cuda")[None], torch.tensor([0, T], dtype=torch.int32, device="cuda")
    tt.cache_append_q4(k, v, slots, kc, vc)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tt.cache_append_q4(k, v, slots, kc, vc)
        a, b = tt.cache_read_q4(kc, vc, table, cu, T, page)
    k.normal_()
    v.normal_()
    slots.copy_(torch.randperm(T))
    g.replay()
    torch.cuda.synchronize()
    want = tt.cache_read_q4(*tt.cache_append_q4(k, v, slots, *tt.cache_alloc_q4(8, hkv, page, D)), table, cu, T, page)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_refusals(tt):
    kc, vc = tt.cache_alloc_q4(4, 2, 16, 64)
    k = torch.randn(5, 2, 64, device="cuda")
    s = torch.arange(5, dtype=torch.int32, device="cuda")
    ok = dict(k=k, v=k, slots=s, k_cache=kc, v_cache=vc)
    tt.cache_append_q4(**ok)
    for kw in (dict(k=k.half(), v=k.half()), dict(k=k.cpu()), dict(k=k[0], v=k[0]), dict(v=k.bfloat16()), dict(v=k[:4]), dict(k=k[:, :1], v=k[:, :1]), dict(k=k.transpose(1, 2)),
               dict(slots=s.long()), dict(slots=s[:4]), dict(slots=torch.zeros(10, dtype=torch.int32, device="cuda")[::2]), dict(slots=s.cpu()), dict(k_cache=kc.int()),
               dict(v_cache=vc[:3]), dict(k_cache=kc.transpose(0, 1), v_cache=vc.transpose(0, 1)), dict(v_cache=kc), dict(k=torch.randn(5, 2, 32, device="cuda"), v=torch.randn(5, 2, 32, device="cuda")),
               dict(k=torch.randn(5, 2, 128, device="cuda"), v=torch.randn(5, 2, 128, device="cuda"))):
        with pytest.raises((ValueError, tt.TTError)):
            tt.cache_append_q4(**{**ok, **kw})
    t, cu = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    ok = dict(k_cache=kc, v_cache=vc, block_table=t, cu_lens=cu, total=5, page_size=16)
    tt.cache_read_q4(**ok)
    for kw in (dict(total=-1), dict(total=2 ** 32), dict(page_size=8), dict(page_size=32), dict(page_size=0), dict(block_table=t.long()), dict(block_table=t[0]), dict(cu_lens=cu[:1]), dict(cu_lens=cu.long()),
               dict(k=torch.empty(5, 2, 64, device="cuda")), dict(v=torch.empty(4, 2, 64, device="cuda").bfloat16()), dict(k_cache=kc.cpu())):
        with pytest.raises(ValueError):
            tt.cache_read_q4(**{**ok, **kw})
    both = torch.empty(5, 2, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="overlap"):
        tt.cache_read_q4(**ok, k=both, v=both)
    for bad in ((4, 2, 8, 64), (4, 2, 24, 64), (4, 2, 16, 96)):
        with pytest.raises(ValueError):
            tt.cache_alloc_q4(*bad)


def test_neighbouring_memory_stays(tt):
    from test_gpu_canary import Guarded
    for T, hkv, D, page, pages in ((1, 1, 64, 16, 1), (37, 3, 128, 48, 1), (128, 2, 64, 16, 8)):
        size = (pages, hkv, page * q4.row_bytes(D))
        kc, vc = Guarded(size, torch.uint8, torch.zeros(size, dtype=torch.uint8)), Guarded(size, torch.uint8, torch.zeros(size, dtype=torch.uint8))
        x = Guarded((T, hkv, D), torch.bfloat16, torch.randn(T, hkv, D))
        tt.cache_append_q4(x.t, x.t, torch.arange(T, dtype=torch.int32, device="cuda"), kc.t, vc.t)
        k, v = Guarded((T, hkv, D), torch.bfloat16), Guarded((T, hkv, D), torch.bfloat16)
        tt.cache_read_q4(kc.t, vc.t, torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([0, T], dtype=torch.int32, device="cuda"), T, page, k=k.t, v=v.t)
        torch.cuda.synchronize()
        assert all(g.intact() for g in (kc, vc, x, k, v))
