"""The 8-bit cache where a call's tokens of one block do not lie together, or share a slot.  That is not allowed, and the block is then unspecified; every other block gets
what the format says, in the same call too."""
import numpy as np
import pytest

import q8_oracle as q8
from test_gpu_cache_q8 import as64, dev, same, spread

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE, HKV = 32, 2
APART = {
    "two blocks in turn": [37, 70] * 50,
    "in turn, a slot each": [x for i in range(16) for x in (32 + i, 64 + i)],
    "one slot again and again": [37] * 100,
    "a run of more than a block": [32 + i % 16 for i in range(70)],
    "others between": [x for i in range(16) for x in (32 + i, -1)],
    "twenty to one slot, then the others": [48] * 20 + [48 + i for i in range(1, 16)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", list(APART))
def test_only_their_blocks_are_unspecified(tt, name, D, dtype):
    apart = APART[name]
    before, behind = list(range(160, 190)), list(range(100, 109))   # sequences of their own in the same call
    slots = np.array(before + apart + behind, np.int32)
    T = len(slots)
    hurt = sorted({s // 16 for s in apart if s >= 0})
    assert not {s // 16 for s in before + behind} & set(hurt)
    pools = [q8.Pool(6, HKV, PAGE, D, 0x33) for _ in range(2)]
    caches = [dev(p.bytes) for p in pools]
    k, v = spread(T, HKV, D, dtype, 1), spread(T, HKV, D, dtype, 2)
    for _ in range(3):
        tt.cache_append_q8(k, v, dev(slots), *caches)
    for p, x, c in zip(pools, (k, v), caches):
        for part in (slice(0, len(before)), slice(T - len(behind), T)):
            for _ in range(3):
                p.write(slots[part], as64(x)[part])
        got = q8.Pool(6, HKV, PAGE, D)
        got.bytes[:] = c.cpu().numpy()
        for a, b in zip(got.parts(), p.parts()):
            at = a.shape[2] // (PAGE // 16)   # rows, or exponents, of a block
            for block in hurt:
                page, j = divmod(block, PAGE // 16)
                a[page, :, at * j:at * j + at] = b[page, :, at * j:at * j + at]
        assert same(got.bytes, p.bytes)
    # written anew from their first rows the blocks are as any
    fresh = np.concatenate([np.arange(16 * b, 16 * b + 16) for b in hurt]).astype(np.int32)
    k, v = spread(len(fresh), HKV, D, dtype, 3), spread(len(fresh), HKV, D, dtype, 4)
    tt.cache_append_q8(k, v, dev(fresh), *caches)
    for p, x, c in zip(pools, (k, v), caches):
        p.write(fresh, as64(x))
        assert same(c.cpu().numpy(), p.bytes)
