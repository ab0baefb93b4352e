"""Decode over the 4-bit cache with queries of every finite size: the head's largest value anywhere in bf16's range."""
import numpy as np
import pytest

from test_gpu_decode_q4 import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [90, 109, 111, 112, 113, 118, 125, -90, -101, -115, -125])
@pytest.mark.parametrize("H,hkv,D", [(4, 2, 128), (12, 1, 64)])
def test_large_and_small_queries_with_moderate_scores(tt, power, H, hkv, D):
    """`scale` takes back what q is larger or smaller by (within the floats that have all their bits); the bounds are those of ordinary queries."""
    scale = 2.0 ** max(-power, -120) * D ** -0.5 if power > 0 else 2.0 ** min(-power, 120) * D ** -0.5
    c = Case([300, 40, 1, 0], H, hkv, D, 16, q_scale=2.0 ** power)
    c.check(*tt.attention_decode_q4(**c.args(), scale=scale), scale)


@pytest.mark.parametrize("power,scale", [(-100, 2.0 ** -60), (-110, 2.0 ** -30), (-126, 2.0 ** -100), (0, 2.0 ** -140)])
def test_scores_that_vanish(tt, power, scale):
    """q and scale both small: all keys count alike, and the places behind the last one do not."""
    c = Case([300, 41, 7, 0], 4, 2, 64, 16, q_scale=2.0 ** power)
    c.check(*tt.attention_decode_q4(**c.args(), scale=scale), scale)
