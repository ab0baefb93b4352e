"""Positions of a shape that could be read in two ways."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_rows_of_positions_without_axes_are_refused(tt):
    """[B, S], the usual layout of position ids, is not taken for [axes, S] of which only the first row would count."""
    B, H, S, D = 3, 2, 5, 8
    x = torch.randn(B, H, S, D, device="cuda")
    freq, _ = tt.rotary_frequencies(D)
    ids = torch.arange(B * S, dtype=torch.int32, device="cuda").view(B, S)
    for call in (tt.rotary_forward, tt.rotary_backward):
        with pytest.raises(ValueError, match="axes"):
            call(x, None, ids, freq)
        with pytest.raises(ValueError, match="axes"):
            call(x, None, ids[:2, None].expand(2, B, S), freq)
        with pytest.raises(ValueError, match="axes"):
            call(x[0].transpose(0, 1), None, ids, freq)
        # one row, and rows with axes, are as they were
        want, _ = call(x, None, ids[0], freq)
        assert torch.equal(want, call(x, None, ids[:1], freq)[0]) and torch.equal(want, call(x, None, ids[:1, None].expand(1, B, S), freq)[0])
        first = torch.zeros(D // 2, dtype=torch.int32, device="cuda")
        assert torch.equal(want, call(x, None, ids, freq, first)[0])
        each, _ = call(x, None, ids[None], freq)
        for b in range(B):
            assert torch.equal(each[b], call(x[b:b + 1], None, ids[b], freq)[0][0])
