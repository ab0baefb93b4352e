"""What the serving calls' results lie on: they can be saved together, and one that is kept does not keep much of what is dropped."""
import io

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("H,lens", [(4, (20, 3)), (16, (200, 500))])
def test_results_of_a_decode_can_be_saved(tt, H, lens):
    page, D = 16, 64
    kc, vc = tt.cache_alloc_q4(80, 2, page, D)
    x = torch.randn(1280, 2, D, device="cuda").bfloat16()
    tt.cache_append_q4(x, x, torch.arange(1280, dtype=torch.int32, device="cuda"), kc, vc)
    table = torch.arange(80, dtype=torch.int32, device="cuda").view(2, 40)
    got = tt.attention_decode_q4(torch.randn(2, H, 1, D, device="cuda").bfloat16(), kc, vc, block_table=table, seq_lens=ints(*lens))
    file = io.BytesIO()
    torch.save(got, file)
    file.seek(0)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.load(file)))
    out, lse = got
    assert out.untyped_storage().nbytes() == out.nbytes and lse.untyped_storage().nbytes() == lse.nbytes


@pytest.mark.parametrize("tokens", [1, 64, 5000, 300000])
def test_kept_lengths_do_not_keep_slots(tt, tokens):
    B, page = 8, 16
    width = (tokens + page - 1) // page + 1
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    free = torch.arange(B * width, dtype=torch.int32, device="cuda")
    step = tt.cache_extend(table, ints(*[0] * B), ints(*[tokens // B + (b < tokens % B) for b in range(B)]), free, ints(B * width), page, tokens)
    for kept in (step.seq_lens, step.n_free):
        assert kept.untyped_storage().nbytes() <= 65536
    assert int(step.cu_new[-1]) == tokens and step.positions.shape == step.slots.shape == (tokens,) and bool((step.slots >= 0).all())
    file = io.BytesIO()
    torch.save(tuple(step), file)
    file.seek(0)
    assert all(torch.equal(a, b) for a, b in zip(step, torch.load(file)))
