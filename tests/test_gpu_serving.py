"""The serving calls as they are used together: prompts in chunks (page tables, rotary positions, the 4-bit cache written and read back, packed
attention), then one token at a time (decode over the cache), requests that leave and others that take their rows and pages."""
import numpy as np
import pytest

import q4_oracle as q4
from test_gpu_decode_q4 import sequence

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Server:
    def __init__(self, tt, rows, pages, page, max_pages, H, hkv, D, seed):
        self.tt, self.page, self.H, self.hkv, self.D = tt, page, H, hkv, D
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.table, self.lens, self.free, self.n_free = ints(rows, max_pages), ints(rows), torch.arange(pages, dtype=torch.int32, device="cuda"), ints(1) + pages
        self.k_cache, self.v_cache = tt.cache_alloc_q4(pages, hkv, page, D)
        self.freq, self.axes = tt.rotary_frequencies(D, sections=(D // 8, D // 8, D // 4), cyclic=True)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.held = [[np.zeros((0, hkv, D)), np.zeros((0, hkv, D))] for _ in range(rows)]   # what each row's cache stands for

    def step(self, new):
        """`new` tokens of each row through the projections' place (random), positions, cache -> (cache step, q)."""
        tt, T = self.tt, int(sum(new))
        step = tt.cache_extend(self.table, self.lens, torch.tensor(new, dtype=torch.int32, device="cuda"), self.free, self.n_free, self.page, T + 5)
        self.lens, self.n_free = step.seq_lens, step.n_free
        rows = torch.randn(T + 5, self.H + 2 * self.hkv, self.D, generator=self.gen, device="cuda").bfloat16()   # one projection's rows
        q, k = rows[:, :self.H], rows[:, self.H:self.H + self.hkv]
        tt.rotary_forward(q, k, step.positions.expand(3, -1), self.freq, self.axes, out_q=q, out_k=k)
        v = rows[:, self.H + self.hkv:]
        tt.cache_append_q4(k, v, step.slots, self.k_cache, self.v_cache)
        cu = step.cu_new.tolist()
        assert np.diff(cu).tolist() == list(new)
        for b in range(len(new)):
            for i, x in enumerate((k, v)):
                values = q4.decode(*q4.encode(x[cu[b]:cu[b + 1]].double().cpu().numpy()))
                self.held[b][i] = np.concatenate([self.held[b][i], values])
        return step, q[:T]

    def release(self, rows):
        done = torch.zeros(len(self.lens), dtype=torch.bool, device="cuda")
        done[rows] = True
        self.lens, self.n_free = self.tt.cache_release(self.table, self.lens, done, self.free, self.n_free, self.page)
        for b in rows:
            self.held[b] = [x[:0] for x in self.held[b]]

    def check(self, b, q, out, lse):
        """One token's heads q [H, D] against row b's cache."""
        q, out, lse, G = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy(), self.H // self.hkv
        for h in range(self.hkv):
            at = slice(h * G, (h + 1) * G)
            o, y, bo, by = sequence(q[at], self.held[b][0][:, h], self.held[b][1][:, h], self.D ** -0.5)
            assert (np.abs(out[at] - o) <= bo).all() and ((lse[at] == y) | (np.abs(lse[at] - y) <= by)).all()


@pytest.mark.parametrize("H,hkv,D,page", [(8, 2, 128, 16), (6, 6, 64, 48)])
def test_prompts_then_tokens(tt, H, hkv, D, page):
    s = Server(tt, 4, 400 // page, page, 200 // page, H, hkv, D, 7)
    G = H // hkv
    for chunk in ([33, 0, 7, 64], [1, 50, 20, 0], [30, 20, 0, 5]):
        step, q = s.step(chunk)
        # the chunk's queries against all that is cached, causal: packed attention over the values read back
        lens = s.lens.tolist()
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        k, v = tt.cache_read_q4(s.k_cache, s.v_cache, s.table, cu, int(sum(lens)), page)
        at = 0
        for b, n in enumerate(lens):
            for x, held in ((k, s.held[b][0]), (v, s.held[b][1])):
                assert np.array_equal(x[at:at + n].double().cpu().numpy(), held)
            at += n
        # sequences without new tokens have keys but no queries
        out, lse = tt.attention_forward_varlen(q.contiguous(), k, v, step.cu_new, cu, max(chunk), max(lens), causal=True)
        at = 0
        for b, n in enumerate(chunk):
            for i in range(n):
                keys = lens[b] - n + i + 1
                for h in range(hkv):
                    heads = slice(h * G, (h + 1) * G)
                    o, _, _, _ = sequence(q[at + i, heads].double().cpu().numpy(), s.held[b][0][:keys, h], s.held[b][1][:keys, h], D ** -0.5)
                    assert np.abs(out[at + i, heads].double().cpu().numpy() - o).max() <= 2e-2   # bf16 attention's bound
            at += n
    for token in range(12):
        if token == 5:
            s.release([0, 3])
        new = [1, 1, 1, 1] if token != 8 else [0, 1, 3, 1]
        step, q = s.step(new)
        last = (step.cu_new[1:] - 1).clamp_min(0).long()
        heads = q[last].unsqueeze(2).contiguous()
        out, lse = tt.attention_decode_q4(heads, s.k_cache, s.v_cache, block_table=s.table, seq_lens=s.lens)
        for b in range(4):
            s.check(b, heads[b, :, 0], out[b, :, 0], lse[b, :, 0])
    assert int(s.n_free) + sum(-(-int(n) // page) for n in s.lens) == 400 // page


def test_captured_token_step(tt):
    """A decode step as one graph, replayed with its own state: lengths, table, cache and free list go on from where they are."""
    B, H, hkv, D, page = 3, 4, 2, 64, 16
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")

    def make():
        table, lens, free, n_free = torch.zeros(B, 8, dtype=torch.int32, device="cuda"), ints([0] * B), torch.arange(30, dtype=torch.int32, device="cuda"), ints([30])
        return [table, lens, free, n_free, *tt.cache_alloc_q4(30, hkv, page, D)]

    freq, _ = tt.rotary_frequencies(D)
    one = ints([1] * B)

    def step(state, rows):
        table, lens, free, n_free, kc, vc = state
        new = tt.cache_extend(table, lens, one, free, n_free, page, B)
        q, k = tt.rotary_forward(rows[:, :H], rows[:, H:H + hkv], new.positions, freq)
        tt.cache_append_q4(k, rows[:, H + hkv:], new.slots, kc, vc)
        out, lse = tt.attention_decode_q4(q.unsqueeze(2), kc, vc, block_table=table, seq_lens=new.seq_lens)
        lens.copy_(new.seq_lens)
        n_free.copy_(new.n_free)
        return out, lse

    rows = torch.randn(B, H + 2 * hkv, D, device="cuda").bfloat16()
    eager, captured = make(), make()
    step(make(), rows)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(captured, rows)
    for i in range(40):
        rows.copy_(torch.randn(rows.shape, device="cuda"))
        want = step(eager, rows)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))
    assert eager[1].tolist() == [40] * B


def test_results_that_share_an_allocation(tt):
    """Short results may lie in one allocation: apart from each other, contiguous, and each usable when the other is gone."""
    import gc
    for T, D in ((1, 64), (3, 50), (40, 128), (5000, 128)):
        q, k = torch.randn(T, 3, D, device="cuda").bfloat16(), torch.randn(T, 1, D, device="cuda").bfloat16()
        freq, _ = tt.rotary_frequencies(D)
        pos = torch.arange(T, dtype=torch.int32, device="cuda")
        a, b = tt.rotary_forward(q, k, pos, freq)
        assert a.is_contiguous() and b.is_contiguous() and a.shape == q.shape and b.shape == k.shape and a.data_ptr() % 16 == b.data_ptr() % 16 == 0
        want = tt.rotary_forward(k, None, pos, freq)[0]
        a.fill_(7)
        assert torch.equal(b, want)
        del a
        gc.collect()
        other = torch.full((T * 4, D), 3.0, device="cuda").bfloat16()
        assert torch.equal(b, want) and (other == 3).all()
    kc, vc = tt.cache_alloc_q4(3, 1, 16, 64)
    x = torch.randn(20, 1, 64, device="cuda").bfloat16()
    tt.cache_append_q4(x, x, torch.arange(20, dtype=torch.int32, device="cuda"), kc, vc)
    table, lens = torch.arange(3, dtype=torch.int32, device="cuda")[None], torch.tensor([20], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    k, v = tt.cache_read_q4(kc, vc, table, cu, 20, 16)
    assert torch.equal(k, v) and k.is_contiguous() and v.is_contiguous()
    k.fill_(7)
    assert torch.equal(v, tt.cache_read_q4(kc, vc, table, cu, 20, 16)[0]) and not (v == 7).all()
    for H in (1, 3, 17):
        q = torch.randn(1, H, 1, 64, device="cuda").bfloat16()
        out, lse = tt.attention_decode_q4(q, kc, vc, block_table=table, seq_lens=lens)
        mine, mine_lse = tt.attention_decode_q4(q, kc, vc, block_table=table, seq_lens=lens, out=torch.empty_like(q), lse=torch.empty(1, H, 1, device="cuda"))
        assert torch.equal(out, mine) and torch.equal(lse, mine_lse) and lse.shape == (1, H, 1) and lse.dtype == torch.float32
        out.fill_(5)
        assert torch.equal(lse, mine_lse)
        lse.fill_(5)
        assert (out == 5).all()
