"""Page tables on the GPU against a loop over the requests: every output of every size equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def cols(n, page):
    return -(-n // page)


def extend_oracle(table, lens, new, free, n_free, page, max_tokens):
    table, B, width = table.copy(), len(lens), table.shape[1]
    n_free = min(max(n_free, 0), len(free))
    left, tokens, lens_out, cu, closed = n_free, 0, lens.copy(), [0], False
    slots, positions = np.full(max_tokens, -1, np.int32), np.zeros(max_tokens, np.int32)
    for b in range(B):
        n, m = int(lens[b]), int(new[b])
        if n >= 0 and m >= 0 and n + m <= width * page and not closed:
            need = cols(n + m, page) - cols(n, page)
            if tokens + m > max_tokens or need > left:
                closed = True
            else:
                for j in range(need):
                    left -= 1
                    table[b, cols(n, page) + j] = free[left]
                for i in range(m):
                    p = table[b, (n + i) // page]
                    slots[tokens] = p * page + (n + i) % page if p >= 0 else -1
                    positions[tokens] = n + i
                    tokens += 1
                lens_out[b] = n + m
        cu.append(tokens)
    return table, lens_out, np.array([left], np.int32), np.array(cu, np.int32), slots, positions


def release_oracle(table, lens, done, free, n_free, page):
    free, lens_out, n_free = free.copy(), lens.copy(), min(max(n_free, 0), len(free))
    for b in range(len(lens)):
        if done[b]:
            for j in range(min(table.shape[1], cols(max(int(lens[b]), 0), page))):
                if n_free < len(free):
                    free[n_free] = table[b, j]
                    n_free += 1
            lens_out[b] = 0
    return free, lens_out, np.array([n_free], np.int32)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def make(rng, B, page, width, longest, most):
    lens = rng.integers(0, longest + 1, B).astype(np.int32)
    new = rng.integers(0, most + 1, B).astype(np.int32)
    pages = rng.permutation(B * width + 50).astype(np.int32)
    table = np.full((B, width), -7, np.int32)
    at = 0
    for b in range(B):
        n = min(width, cols(int(lens[b]), page))
        table[b, :n] = pages[at:at + n]
        at += n
    return table, lens, new, pages[at:].copy()


def check_extend(tt, table, lens, new, free, n_free, page, max_tokens, out=None):
    want = extend_oracle(table, lens, new, free, n_free, page, max_tokens)
    t, f = dev(table), dev(free)
    step = tt.cache_extend(t, dev(lens), dev(new), f, dev(np.array([n_free], np.int32)), page, max_tokens, out=out)
    got = (t,) + tuple(step)
    for name, a, b in zip(("table", "lens", "n_free", "cu", "slots", "positions"), got, want):
        assert np.array_equal(a.cpu().numpy(), b), name
    assert np.array_equal(f.cpu().numpy(), free)
    return step


@pytest.mark.parametrize("B,page,width,longest,most", [
    (1, 16, 4, 0, 1), (1, 1, 9, 4, 5), (3, 16, 8, 60, 40), (64, 64, 40, 2000, 1), (37, 7, 50, 300, 20), (255, 16, 9, 100, 44), (256, 32, 6, 150, 1),
    (257, 16, 9, 100, 17), (1000, 128, 3, 256, 100), (1024, 16, 2, 16, 16), (1025, 16, 3, 30, 15), (5000, 16, 2, 20, 3), (16384, 8, 2, 9, 1)])
def test_extend(tt, B, page, width, longest, most):
    rng = np.random.default_rng(B * 31 + page)
    table, lens, new, free = make(rng, B, page, width, longest, most)
    total = int(new.sum())
    need = sum(cols(int(a + b), page) - cols(int(a), page) for a, b in zip(lens, new))
    for n_free, tokens in ((len(free), total), (len(free), total + 33), (need, total), (max(0, need - 1), total + 1), (need // 2, total), (len(free), max(0, total - 1)),
                           (0, total), (-5, total), (len(free) + 99, total), (len(free), 0)):
        check_extend(tt, table, lens, new, free, n_free, page, tokens)


def test_extend_passes_over_what_cannot_be_served(tt):
    rng = np.random.default_rng(5)
    table, lens, new, free = make(rng, 40, 16, 6, 60, 30)
    lens[3], new[7], lens[11], new[12], lens[20], new[20] = -1, -4, 97, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1
    lens[15], new[15] = 96, 0      # a full row without new tokens
    lens[16], new[16] = 96, 1      # and one with
    check_extend(tt, table, lens, new, free, len(free), 16, 2000)
    # new tokens on a page whose entry is negative have no slot
    lens[0], new[0] = 20, 30
    table[0, 1] = -3
    step = check_extend(tt, table, lens, new, free, len(free), 16, 2000)
    assert (step.slots[:12] == -1).all() and (step.slots[12:30] >= 0).all()


@pytest.mark.parametrize("B,page,width,longest", [(1, 16, 3, 40), (50, 64, 30, 1900), (300, 16, 20, 330), (1025, 8, 4, 40), (16384, 16, 2, 32)])
def test_release(tt, B, page, width, longest):
    rng = np.random.default_rng(B)
    table, lens, _, spare = make(rng, B, page, width, longest, 0)
    lens[0] = -2
    for share, capacity, n_free in ((0.0, 9999999, 3), (0.5, 9999999, 0), (1.0, 9999999, 7), (0.7, len(spare) + 5, len(spare)), (1.0, 10, 10), (0.5, 9999999, -4)):
        done = rng.random(B) < share
        free = np.concatenate([spare, np.full(min(capacity, len(spare) + B * width) - len(spare), -9, np.int32)]) if capacity > len(spare) else spare[:capacity]
        want = release_oracle(table, lens, done, free, n_free, page)
        t, f = dev(table), dev(free)
        for d in (dev(done), dev(done).to(torch.uint8) * 255):
            f.copy_(dev(free))
            got_lens, got_free = tt.cache_release(t, dev(lens), d, f, dev(np.array([n_free], np.int32)), page)
            for a, b in zip((f, got_lens, got_free), want):
                assert np.array_equal(a.cpu().numpy(), b)
        assert np.array_equal(t.cpu().numpy(), table)


def test_pages_go_round(tt):
    """Requests come, grow and leave for 60 steps: no page belongs to two requests, none is lost."""
    rng = np.random.default_rng(1)
    B, page, width, pool = 24, 16, 12, 140
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    lens, free, n_free = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.arange(pool, dtype=torch.int32, device="cuda"), torch.tensor([pool], dtype=torch.int32, device="cuda")
    out = None
    for step in range(60):
        new = torch.from_numpy(rng.integers(0, 20, B).astype(np.int32)).cuda()
        a = tt.cache_extend(table, lens, new, free, n_free, page, B * 20, out=out)
        out = (lens, n_free) + tuple(a[2:]) if step else None   # the buffers of the step before
        lens, n_free = a.seq_lens, a.n_free
        done = torch.from_numpy(rng.random(B) < 0.1).cuda() | (lens > width * page - 20)
        lens, n_free = tt.cache_release(table, lens, done, free, n_free, page)
        held = [table[b, :cols(int(lens[b]), page)].tolist() for b in range(B)]
        assert sorted(sum(held, []) + free[:int(n_free)].tolist()) == list(range(pool))


def test_captured_step_replays_on_new_lengths(tt):
    rng = np.random.default_rng(9)
    table, lens, new, free = make(rng, 33, 16, 8, 60, 30)
    t, l, m, f, n = dev(table), dev(lens), dev(new), dev(free), dev(np.array([len(free)], np.int32))
    out = tt.cache_extend(t, l, m, f, n, 16, 1000)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tt.cache_extend(t, l, m, f, n, 16, 1000, out=out)
    for seed in (1, 2):
        table, lens, new, free = make(np.random.default_rng(seed), 33, 16, 8, 60, 30)
        free = free[:len(f)] if len(free) >= len(f) else np.concatenate([free, np.full(len(f) - len(free), -1, np.int32)])
        n_free = min(60, len(f))
        for a, b in ((t, table), (l, lens), (m, new), (f, free)):
            a.copy_(torch.from_numpy(b))
        n.fill_(n_free)
        g.replay()
        want = extend_oracle(table, lens, new, free, n_free, 16, 1000)
        for a, b in zip((t,) + tuple(out), want):
            assert np.array_equal(a.cpu().numpy(), b)


def test_refusals(tt):
    i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    t = torch.zeros(4, 8, dtype=torch.int32, device="cuda")
    ok = (t, i(4), i(4), i(9), i(1), 16, 5)
    tt.cache_extend(*ok)
    for at, bad in ((0, t[:, :4]), (0, t.long()), (0, t[0]), (1, i(5)), (1, i(8)[::2]), (2, i(4).float()), (3, i(9).cpu()), (4, i(2)), (5, 0), (5, 2 ** 32 + 16), (6, -1), (6, 2 ** 32)):
        with pytest.raises(ValueError):
            tt.cache_extend(*(bad if k == at else x for k, x in enumerate(ok)))
    good = tt.cache_extend(*ok)
    for bad in (good[:4], list(good), good._replace(slots=i(4)), good._replace(cu_new=i(4)), good._replace(seq_lens=ok[1]), good._replace(n_free=i(1).long())):
        with pytest.raises(ValueError):
            tt.cache_extend(*ok, out=bad)
    with pytest.raises(TypeError):
        tt.cache_extend(*ok[:5], [16], 5)
    with pytest.raises(ValueError):
        tt.cache_release(t, i(4), i(4), i(9), i(1), 16)
    with pytest.raises(ValueError):
        tt.cache_release(t, i(4), i(4).bool(), i(9), i(1), 16, out=(i(3), i(1)))
