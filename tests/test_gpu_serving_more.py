"""The calls between a projection and its attention as they are used together: page tables, normed and turned heads, the 8-bit cache written, read back
and decoded; and the same over the 16-bit cache, where norm, rotation and cache are one call."""
import numpy as np
import pytest

import norm_rotary_oracle as nr
import q8_oracle as q8
from test_gpu_decode_q8 import sequence

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Server:
    def __init__(self, tt, rows, pages, page, max_pages, H, hkv, D, seed, bits):
        self.tt, self.page, self.H, self.hkv, self.D, self.bits = tt, page, H, hkv, D, bits
        self.table, self.lens = torch.zeros(rows, max_pages, dtype=torch.int32, device="cuda"), ints([0] * rows)
        self.free, self.n_free = torch.arange(pages, dtype=torch.int32, device="cuda"), ints([pages])
        if bits == 8:
            self.k_cache, self.v_cache = tt.cache_alloc_q8(pages, hkv, page, D)
            self.pools = [q8.Pool(pages, hkv, page, D) for _ in range(2)]
        else:
            self.k_cache, self.v_cache = (torch.zeros(pages, hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.freq, _ = tt.rotary_frequencies(D)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.w = [(1 + 0.2 * torch.randn(D, generator=self.gen, device="cuda")).bfloat16() for _ in range(2)]

    def step(self, new):
        """`new` tokens of each row through the projections' place (random), norm, positions, cache -> (cache step, q)."""
        tt, T = self.tt, int(sum(new))
        step = tt.cache_extend(self.table, self.lens, ints(new), self.free, self.n_free, self.page, T + 5)
        self.lens, self.n_free = step.seq_lens, step.n_free
        rows = torch.randn(T + 5, self.H + 2 * self.hkv, self.D, generator=self.gen, device="cuda").bfloat16()   # one projection's rows
        q, k, v = rows[:, :self.H], rows[:, self.H:self.H + self.hkv], rows[:, self.H + self.hkv:]
        if self.bits == 8:
            tt.norm_rotary_forward(q, k, *self.w, step.positions, self.freq, out_q=q, out_k=k)
            tt.cache_append_q8(k, v, step.slots, self.k_cache, self.v_cache)
            for pool, x, got in zip(self.pools, (k, v), (self.k_cache, self.v_cache)):
                pool.write(step.slots.cpu().numpy(), x.double().cpu().numpy())
                assert np.array_equal(got.cpu().numpy(), pool.bytes)
            return step, q[:T]
        before = k.clone(), v.clone()
        q = tt.cache_append_rotary(q, k, v, step.slots, step.positions, self.freq, self.k_cache, self.v_cache, q_weight=self.w[0], k_weight=self.w[1])
        assert torch.equal(k, before[0])
        return step, q[:T]

    def held(self, b):
        """Row b's keys, values [n, hkv, D] and its values' exponents, 64 bits."""
        n, table = int(self.lens[b]), self.table[b].cpu().numpy()
        if self.bits == 8:
            return self.pools[0].rows(table, n), self.pools[1].rows(table, n), self.pools[1].exponents(table, n)
        at = torch.arange(n, device="cuda")
        page = self.table[b, at // self.page].long()
        return (*(x[page, :, at % self.page].double().cpu().numpy() for x in (self.k_cache, self.v_cache)), np.zeros((n, self.hkv)))

    def check(self, b, q, out, lse, bound=None):
        k, v, ev = self.held(b)
        q, out, lse, G = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy(), self.H // self.hkv
        for h in range(self.hkv):
            at = slice(h * G, (h + 1) * G)
            o, y, bo, by = sequence(q[at], k[:, h], v[:, h], ev[:, h], self.D ** -0.5)
            if bound is not None:
                bo, by = bound, bound
            assert (np.abs(out[at] - o) <= bo).all() and ((lse[at] == y) | (np.abs(lse[at] - y) <= by)).all()


@pytest.mark.parametrize("H,hkv,D,page", [(8, 2, 128, 16), (6, 6, 64, 48)])
def test_prompts_then_tokens_over_8_bits(tt, H, hkv, D, page):
    s = Server(tt, 4, 400 // page, page, 200 // page, H, hkv, D, 7, 8)
    G = H // hkv
    for chunk in ([33, 0, 7, 64], [1, 50, 20, 0], [30, 20, 0, 5]):
        step, q = s.step(chunk)
        lens = s.lens.tolist()
        cu = ints(np.concatenate([[0], np.cumsum(lens)]).tolist())
        k, v = tt.cache_read_q8(s.k_cache, s.v_cache, s.table, cu, int(sum(lens)), page)
        at = 0
        for b, n in enumerate(lens):
            for x, held in zip((k, v), s.held(b)):
                assert np.array_equal(x[at:at + n].double().cpu().numpy(), held)
            at += n
        out, lse = tt.attention_forward_varlen(q.contiguous(), k, v, step.cu_new, cu, max(chunk), max(lens), causal=True)
        at = 0
        for b, n in enumerate(chunk):
            hk, hv, ev = s.held(b)
            for i in range(n):
                keys = lens[b] - n + i + 1
                for h in range(hkv):
                    heads = slice(h * G, (h + 1) * G)
                    o, _, _, _ = sequence(q[at + i, heads].double().cpu().numpy(), hk[:keys, h], hv[:keys, h], ev[:keys, h], D ** -0.5)
                    assert np.abs(out[at + i, heads].double().cpu().numpy() - o).max() <= 2e-2   # bf16 attention's bound
            at += n
    for token in range(20):
        new = [1, 1, 1, 1] if token != 8 else [0, 1, 3, 1]
        step, q = s.step(new)
        heads = q[(step.cu_new[1:] - 1).clamp_min(0).long()].unsqueeze(2).contiguous()
        out, lse = tt.attention_decode_q8(heads, s.k_cache, s.v_cache, block_table=s.table, seq_lens=s.lens)
        for b in range(4):
            s.check(b, heads[b, :, 0], out[b, :, 0], lse[b, :, 0])


@pytest.mark.parametrize("H,hkv,D,page", [(8, 2, 128, 16), (6, 6, 64, 64)])
def test_prompts_then_tokens_over_16_bits(tt, H, hkv, D, page):
    s = Server(tt, 3, 600 // page, page, 200 // page, H, hkv, D, 9, 16)
    for chunk in ([33, 0, 70], [1, 50, 20]):
        s.step(chunk)
    for token in range(10):
        step, q = s.step([1, 1, 1])
        heads = q.unsqueeze(2)
        out, lse = tt.attention_decode_paged(heads, s.k_cache, s.v_cache, block_table=s.table, seq_lens=s.lens)
        for b in range(3):
            s.check(b, heads[b, :, 0], out[b, :, 0], lse[b, :, 0], 2e-2)   # bf16 attention's bound


def test_prompt_through_packed_attention(tt):
    """A prompt's first chunk: the turned keys go to the cache and, packed, to the attention over the chunk itself, with equal bits."""
    T, H, hkv, D, page = 150, 8, 2, 128, 64
    s = Server(tt, 1, 4, page, 4, H, hkv, D, 3, 16)
    step = tt.cache_extend(s.table, s.lens, ints([T]), s.free, s.n_free, page, T)
    rows = torch.randn(T, H + 2 * hkv, D, device="cuda").bfloat16()
    q, k, v = rows[:, :H], rows[:, H:H + hkv], rows[:, H + hkv:]
    packed_k = torch.empty(T, hkv, D, device="cuda", dtype=torch.bfloat16)
    turned = tt.cache_append_rotary(q, k, v, step.slots, step.positions, s.freq, s.k_cache, s.v_cache, q_weight=s.w[0], k_weight=s.w[1], out_k=packed_k)
    out, _ = tt.attention_forward_varlen(turned, packed_k, v.contiguous(), step.cu_new, step.cu_new, T, T, causal=True)
    last = turned[-1:].unsqueeze(2)
    again, _ = tt.attention_decode_paged(last, s.k_cache, s.v_cache, block_table=s.table, seq_lens=step.seq_lens)
    assert (out[-1].float() - again[0, :, 0].float()).abs().max() <= 2e-2   # two kernels, each within bf16 attention's bound of 1e-2 or so
    at = step.slots.long()
    assert torch.equal(s.k_cache[at // page, :, at % page], packed_k) and torch.equal(s.v_cache[at // page, :, at % page], v)


@pytest.mark.parametrize("bits", [8, 16])
def test_captured_token_step(tt, bits):
    """A decode step as one graph, replayed with its own state: lengths, table, cache and free list go on from where they are."""
    B, H, hkv, D, page = 3, 4, 2, 64, 16

    def make():
        cache = tt.cache_alloc_q8(30, hkv, page, D) if bits == 8 else [torch.zeros(30, hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        return [torch.zeros(B, 8, dtype=torch.int32, device="cuda"), ints([0] * B), torch.arange(30, dtype=torch.int32, device="cuda"), ints([30]), *cache]

    freq, _ = tt.rotary_frequencies(D)
    one = ints([1] * B)
    w = torch.rand(D, device="cuda") + 0.5

    def step(state, rows):
        table, lens, free, n_free, kc, vc = state
        new = tt.cache_extend(table, lens, one, free, n_free, page, B)
        q, k, v = rows[:, :H], rows[:, H:H + hkv], rows[:, H + hkv:]
        if bits == 8:
            q, k = tt.norm_rotary_forward(q, k, w, w, new.positions, freq)
            tt.cache_append_q8(k, v, new.slots, kc, vc)
            out, lse = tt.attention_decode_q8(q.unsqueeze(2), kc, vc, block_table=table, seq_lens=new.seq_lens)
        else:
            q = tt.cache_append_rotary(q, k, v, new.slots, new.positions, freq, kc, vc, q_weight=w, k_weight=w)
            out, lse = tt.attention_decode_paged(q.unsqueeze(2), kc, vc, block_table=table, seq_lens=new.seq_lens)
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
        rows.copy_(torch.randn(rows.shape, device="cuda") * (1 + i % 7))
        want = step(eager, rows)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))
    assert eager[1].tolist() == [40] * B


def test_training_step_as_a_graph(tt):
    """Normed and turned heads, attention and the way back, captured and replayed: gradients of heads and weights equal the eager calls'."""
    B, H, hkv, S, D = 1, 4, 2, 96, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    q, k, v, dout, wq, wk = new(B, H, S, D), new(B, hkv, S, D), new(B, hkv, S, D), new(B, H, S, D), new(D), new(D)
    freq, _ = tt.rotary_frequencies(D)
    pos = torch.arange(S, dtype=torch.int32, device="cuda")

    def step():
        a, b = tt.norm_rotary_forward(q, k, wq, wk, pos, freq)
        out, lse = tt.attention_forward(a, b, v, causal=True)
        da, db, dv = tt.attention_backward(a, b, v, out, lse, dout, causal=True)
        return (out, dv) + tt.norm_rotary_backward(da, db, q, k, wq, wk, pos, freq)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        for x in (q, k, v, dout, wq, wk):
            x.normal_(generator=g)
        graph.replay()
        # (dq of the attention is summed in no fixed order where its single pass is taken)
        for a, b in zip(got, step()):
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(b.float().abs().max()))
    # against the formula, from what the attention handed back
    a, b = tt.norm_rotary_forward(q, k, wq, wk, pos, freq)
    out, lse = tt.attention_forward(a, b, v, causal=True)
    da, db, _ = tt.attention_backward(a, b, v, out, lse, dout, causal=True)
    t = nr.angles(pos.cpu().numpy()[None], freq.tolist(), None)
    for x, dz, w, dx, dw in zip((q, k), (da, db), (wq, wk), *[iter(tt.norm_rotary_backward(da, db, q, k, wq, wk, pos, freq)[i:i + 2]) for i in (0, 2)]):
        want, ex, want_w, ew = nr.backward(*(y.double().cpu().numpy() for y in (dz, x, w)), t)
        for y, z, e in ((dx, want, ex), (dw, want_w, ew)):
            ok, worst = nr.within(y.double().cpu().numpy(), z, e, torch.finfo(y.dtype).eps)
            assert ok, worst
