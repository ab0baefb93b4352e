"""Normed heads with rotary positions, and appending with them, where each CTA goes through several tiles of tokens: to the bit what the same rows give in calls
so short that no CTA has a second token, and some rows against 64 bits by the bounds of norm_rotary_oracle."""
import numpy as np
import pytest

import norm_rotary_oracle as nr
from test_gpu_norm_rotary import host, near, weights

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PIECE = 100   # tokens: fewer than a B200 has SMs


def tokens(heads, D, dtype, per_sm=3, tiles=2.3):
    """Tokens for at least two tiles to a CTA: a tile is at most 28 turns of 256 threads with two accesses of 16 bytes each."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert PIECE < sms
    return int(tiles * per_sm * sms * 28 * 256 * 2 * (128 // torch.finfo(dtype).bits) / (heads * D)) + 7


def some(T, seed=0):
    """Tokens to look at: the first, the last, and others."""
    return np.unique(np.concatenate(([0, 1, T - 1], np.random.default_rng(seed).integers(0, T, 30))))


def check(tt, q, k, pos, freq, axes, interleaved, wtype, back):
    """q, k packed [T, heads, D], pos [A, T]"""
    T, D = q.shape[0], q.shape[-1]
    wq, wk = weights(D, wtype, 1), weights(D, wtype, 2)
    how = dict(axes=axes, interleaved=interleaved)
    got = tt.norm_rotary_forward(q, k, wq, wk, pos, freq, **how)
    g = [torch.randn(x.shape, device="cuda").to(x.dtype) for x in (q, k)] if back else None
    dx = tt.norm_rotary_backward(*g, q, k, wq, wk, pos, freq, **how) if back else None
    for s in range(0, T, PIECE):
        at = slice(s, min(s + PIECE, T))
        piece = tt.norm_rotary_forward(q[at], k[at], wq, wk, pos[:, at], freq, **how)
        assert all(torch.equal(x[at], y) for x, y in zip(got, piece)), s
        if back:
            piece = tt.norm_rotary_backward(g[0][at], g[1][at], q[at], k[at], wq, wk, pos[:, at], freq, **how)
            assert all(torch.equal(x[at], y) for x, y in zip(dx[:2], piece[:2])), s
    at = some(T)
    t = nr.angles(pos.cpu().numpy()[:, at], freq.tolist(), axes.tolist() if axes is not None else None)[:, None]
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        near(got[i][at], *nr.forward(host(x[at]), host(w), t, interleaved))
        if back:
            want, bound, _, _ = nr.backward(host(g[i][at]), host(x[at]), host(w), t, interleaved)
            near(dx[i][at], want, bound)


# heads, channels, turned ones: bf16 rows with one unit to a lane (all channels of few heads turned, and heads of 64), with two, rows that are not whole, narrow accesses
@pytest.mark.parametrize("H,Hkv,D,R,dtype,back", [(8, 2, 128, 128, torch.bfloat16, True), (32, 8, 64, 32, torch.bfloat16, True), (32, 8, 128, 128, torch.bfloat16, False), (12, 4, 128, 16, torch.bfloat16, False),
                                                  (6, 3, 256, 128, torch.bfloat16, False), (5, 5, 80, 80, torch.bfloat16, True), (16, 4, 80, 20, torch.bfloat16, False), (7, 1, 96, 24, torch.bfloat16, False),
                                                  (8, 8, 64, 32, torch.float32, True), (9, 3, 128, 128, torch.float32, False), (3, 2, 65, 12, torch.float32, False)])
def test_packed_and_fused(tt, H, Hkv, D, R, dtype, back):
    T = tokens(H + Hkv, D, dtype)
    torch.manual_seed(D + H)
    rows = torch.randn(T, H + 2 * Hkv, D, device="cuda").to(dtype)
    freq, axes = tt.rotary_frequencies(R, sections=(R // 2 - R // 4, R // 4) if R > 2 else None)
    pos = torch.randint(0, 100000, (2, T), device="cuda", dtype=torch.int32)
    check(tt, rows[:, :H], rows[:, H:H + Hkv], pos, freq, axes, H % 2 == 1, torch.float32 if H % 3 else dtype, back)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_dense(tt, dtype):
    """Batch entries that end inside a CTA's share and inside a tile."""
    B, H, D = 5, 12, 128
    S = tokens(H, D, dtype) // B + 3
    x = torch.randn(B, H, S, D, device="cuda").to(dtype)
    freq, _ = tt.rotary_frequencies(D)
    pos = torch.randint(0, 100000, (1, B, S), device="cuda", dtype=torch.int32)
    w = weights(D, torch.float32, 1)
    got, _ = tt.norm_rotary_forward(x, None, w, None, pos, freq)
    step = PIECE // B
    for s in range(0, S, step):
        at = slice(s, min(s + step, S))
        assert torch.equal(got[:, :, at], tt.norm_rotary_forward(x[:, :, at], None, w, None, pos[:, :, at], freq)[0]), s
    at = some(S)
    t = nr.angles(pos.cpu().numpy()[:, :, at], freq.tolist(), None)[:, None]
    near(got[:, :, at], *nr.forward(host(x[:, :, at]), host(w), t))


@pytest.mark.parametrize("H,Hkv,D,R,page,dtype,normed", [(32, 8, 128, 128, 64, torch.bfloat16, True), (6, 2, 64, 64, 16, torch.bfloat16, False), (0, 4, 128, 32, 48, torch.bfloat16, True),
                                                        (8, 8, 64, 20, 16, torch.bfloat16, True), (4, 4, 128, 64, 7, torch.float32, True), (0, 2, 64, 64, 128, torch.float32, False)])
def test_append(tt, H, Hkv, D, R, page, dtype, normed):
    T = tokens(H + 2 * Hkv, D, dtype, per_sm=2 if D % 16 == 0 and R % 16 == 0 else 3)
    torch.manual_seed(D + H)
    rows = torch.randn(T, H + 2 * Hkv, D, device="cuda").to(dtype)
    q, k, v = rows[:, :H] if H else None, rows[:, H:H + Hkv], rows[:, H + Hkv:]
    pages = T // page + 2
    slots = torch.randperm(pages * page, device="cuda")[:T].int()
    slots[5::97] = -1
    pos = torch.randint(0, 100000, (T,), device="cuda", dtype=torch.int32)
    freq, _ = tt.rotary_frequencies(R)
    w = [weights(D, torch.float32, 1) if H and normed else None, weights(D, torch.float32, 2) if normed else None]
    pools = [torch.zeros(2, pages, Hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    also = torch.empty(T, Hkv, D, device="cuda", dtype=torch.bfloat16)
    how = dict(q_weight=w[0], k_weight=w[1])
    got = tt.cache_append_rotary(q, k, v, slots, pos, freq, pools[0][0], pools[1][0], out_k=also, **how)
    for s in range(0, T, PIECE):
        at = slice(s, min(s + PIECE, T))
        mine = torch.empty_like(also[at])
        piece = tt.cache_append_rotary(q[at] if H else None, k[at], v[at], slots[at], pos[at], freq, pools[0][1], pools[1][1], out_k=mine, **how)
        assert torch.equal(also[at], mine) and (not H or torch.equal(got[at], piece)), s
    assert all(torch.equal(p[0], p[1]) for p in pools)
    kept = (slots >= 0).nonzero()[:, 0]
    at = slots[kept].long()
    assert torch.equal(pools[0][0][at // page, :, at % page], also[kept]) and torch.equal(pools[1][0][at // page, :, at % page], v[kept].bfloat16())
    at = some(T)
    t = nr.angles(pos.cpu().numpy()[None, at], freq.tolist(), None)[:, None]
    near(also[at], *nr.forward(host(k[at]), host(w[1]) if normed else None, t))
    if H:
        near(got[at], *nr.forward(host(q[at]), host(w[0]) if normed else None, t))
