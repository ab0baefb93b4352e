"""The serving calls once more, by bounds of their own: prompt chunks through packed attention over values read back from the 4-bit cache, and what a decode
may give where the cache's unused rows hold anything.

Packed attention's bound per output value: scores as in the decode's (u = 2^-23, (D + 2) u scale sum |q k|), the exponential's 2^-22 and its argument's rounding, both
doubled for the row's sum; probabilities rounded to bf16, half a step of 2^-8 of themselves; sums of n values in steps of 16, (n / 16 + 40) u of sum p |v|;
and the result's rounding, 2^-8 of it."""
import numpy as np
import pytest

from test_gpu_decode_q4 import Case, U, dev
from test_gpu_serving import Server

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def attended(q, k, v, scale):
    """q [G, D], k, v [n, D] -> (out, bound)."""
    n, D = k.shape
    s = q @ k.T * scale
    ds = (D + 2) * U * scale * (np.abs(q) @ np.abs(k).T).max(-1)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    out = p @ v
    rel = 2 * np.expm1(ds) + 2.0 ** -20 + 2.0 ** -8 + (n / 16 + 40) * U
    return out, 1.0625 * rel[:, None] * (p @ np.abs(v)) + 2.0 ** -8 * np.abs(out)


@pytest.mark.parametrize("H,hkv,D,page", [(8, 2, 128, 16), (6, 6, 64, 48), (4, 1, 64, 16)])
def test_prompt_chunks(tt, H, hkv, D, page):
    s = Server(tt, 3, 600 // page, page, 250 // page, H, hkv, D, 11)
    G = H // hkv
    for chunk in ([40, 0, 7], [1, 90, 0], [60, 33, 129]):
        step, q = s.step(chunk)
        lens = s.lens.tolist()
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        k, v = tt.cache_read_q4(s.k_cache, s.v_cache, s.table, cu, int(sum(lens)), page)
        out, _ = tt.attention_forward_varlen(q.contiguous(), k, v, step.cu_new, cu, max(chunk), max(lens), causal=True)
        got, at = out.double().cpu().numpy(), 0
        for b, n in enumerate(chunk):
            for i in range(n):
                keys = lens[b] - n + i + 1
                for h in range(hkv):
                    heads = slice(h * G, (h + 1) * G)
                    want, bound = attended(q[at + i, heads].double().cpu().numpy(), s.held[b][0][:keys, h], s.held[b][1][:keys, h], D ** -0.5)
                    assert (np.abs(got[at + i, heads] - want) <= bound).all(), (b, i, h, float((np.abs(got[at + i, heads] - want) / bound).max()))
            at += n


@pytest.mark.parametrize("lens", [[1, 17, 33, 500], [0, 15, 129, 130], [0, 1, 127, 128]])
@pytest.mark.parametrize("fill", [0xFF, 0xDF, 0x00])
def test_unused_rows_give_nothing(tt, lens, fill):
    """NaN, the largest finite scales and zeros where no sequence has a row: finite results, within the bounds, and -inf for empty sequences alone."""
    c = Case(lens, 8, 2, 128, 64, fill=fill)
    out, lse = tt.attention_decode_q4(**c.args())
    assert torch.isfinite(out).all()
    empty = torch.tensor(lens, device="cuda") == 0
    assert torch.isfinite(lse[~empty]).all() and (lse[empty] == -torch.inf).all() and not out[empty].any()
    c.check(out, lse)
    a = c.args()
    a["seq_lens"] = dev(np.array([max(n - 1, 0) for n in lens], np.int32))   # one key fewer: the last row is unused, too
    c.lens = [max(n - 1, 0) for n in lens]
    c.check(*tt.attention_decode_q4(**a))
