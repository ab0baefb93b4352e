"""Pages given back from tables with negative entries (pages that a sliding window has dropped, say): an entry that is no page does not get on the free list."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def cols(n, page):
    return -(-n // page)


def release_oracle(table, lens, done, free, n_free, page):
    free, n_free = free.copy(), min(max(n_free, 0), len(free))
    for b in np.flatnonzero(done):
        for p in table[b, :cols(max(int(lens[b]), 0), page)]:
            if p >= 0 and n_free < len(free):
                free[n_free] = p
                n_free += 1
    return free, np.where(done, 0, lens).astype(np.int32), np.array([n_free], np.int32)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


@pytest.mark.parametrize("B,page,width,longest", [(1, 16, 1, 16), (1, 16, 5000, 80000), (2, 1, 513, 513), (7, 16, 70, 1000), (50, 64, 30, 1900), (300, 16, 1100, 17600), (1025, 8, 4, 40),
                                                  (16384, 16, 3, 48), (1030, 16, 70, 1120), (16384, 8, 5, 40)])
@pytest.mark.parametrize("share", [0.0, 0.0005, 0.02, 0.5, 1.0])
def test_holes_stay_off_the_list(tt, B, page, width, longest, share):
    rng = np.random.default_rng(B + width)
    table = rng.permutation(B * width).astype(np.int32).reshape(B, width)
    holes = rng.random((B, width)) < share
    table[holes] = -rng.integers(1, 2 ** 31, int(holes.sum())).astype(np.int32)
    lens = rng.integers(0, longest + 1, B).astype(np.int32)
    lens[B // 2] = longest
    for marked, capacity, n_free in ((1.0, B * width + 9, 4), (0.5, B * width, 0), (1.0, B * width // 3 + 2, 2), (0.0, 5, 5)):
        done = rng.random(B) < marked
        done[B // 2] = marked > 0
        free = rng.integers(0, 10 ** 6, capacity).astype(np.int32)
        want = release_oracle(table, lens, done, free, n_free, page)
        reach = n_free + sum(min(width, cols(int(n), page)) for n in lens[done])   # of all entries, if none were left out
        for before in (-2 ** 31, 77):   # what the output for the count held
            t, f = dev(table), dev(free)
            out = (torch.full((B,), -2 ** 31, dtype=torch.int32, device="cuda"), torch.full((1,), before, dtype=torch.int32, device="cuda"))
            got_lens, got_n = tt.cache_release(t, dev(lens), dev(done), f, dev(np.array([n_free], np.int32)), page, out=out)
            assert np.array_equal(got_lens.cpu().numpy(), want[1]) and np.array_equal(got_n.cpu().numpy(), want[2])
            got, n = f.cpu().numpy(), int(got_n)
            assert np.array_equal(got[:n], want[0][:n]) and np.array_equal(got[reach:], free[reach:])
            assert np.array_equal(t.cpu().numpy(), table)


def test_a_window_that_drops_pages(tt):
    """Requests whose oldest pages the server takes back by itself, row by row, before they are released: every page is in one place, and what new requests
    get are pages, with a slot for each of their tokens."""
    page, width, pool, B = 16, 8, 40, 5
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, lens, free, n_free = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), ints([0] * B), torch.arange(pool, dtype=torch.int32, device="cuda"), ints([pool])
    step = tt.cache_extend(table, lens, ints([100, 40, 128, 1, 60]), free, n_free, page, 400)
    lens, n_free = step.seq_lens, step.n_free
    for b, columns in ((0, 3), (2, 5), (4, 4)):   # the first pages of these leave the window
        n = int(n_free)
        free[n:n + columns] = table[b, :columns]
        table[b, :columns] = -1
        n_free = ints([n + columns])
    lens, n_free = tt.cache_release(table, lens, torch.tensor([True, False, True, False, True], device="cuda"), free, n_free, page)
    held = table[1, :3].tolist() + table[3, :1].tolist()
    assert sorted(held + free[:int(n_free)].tolist()) == list(range(pool))
    step = tt.cache_extend(table, lens, ints([128, 0, 128, 0, 128]), free, n_free, page, 400)
    assert (step.slots[:384] >= 0).all() and step.slots[:384].unique().numel() == 384
