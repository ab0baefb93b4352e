"""The 8-bit cache's number format in NumPy, 64 bits: codes by search among all 8-bit floats, exponents by trying them."""
import numpy as np

LOW, HIGH, BIAS, TOP = -40, 40, 64, 448.0
_N = np.arange(256)
with np.errstate(invalid="ignore"):
    CODES = np.where(_N & 128, -1.0, 1.0) * np.where(_N >> 3 & 15, (8 + (_N & 7)) * 2.0 ** ((_N >> 3 & 15) - 10.0), (_N & 7) * 2.0 ** -9)
    CODES[[127, 255]] = np.nan
POSITIVE = CODES[:127]


def nearest(y):
    """Codes of values y: to the nearest, ties to the even code; beyond the largest the largest, NaN 127."""
    y = np.asarray(y, np.float64)
    size = np.where(np.isnan(y), 0, np.minimum(np.abs(y), TOP))
    hi = np.minimum(np.searchsorted(POSITIVE, size), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = POSITIVE[hi] - size, size - POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isnan(y), 127, code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def exponent(x):
    """The smallest e with 448 * 2^e >= every finite |x|, of the last axis and the one before the heads: x [n, hkv, D] -> [hkv]."""
    size = np.abs(np.where(np.isfinite(x), x, 0.0)).max((0, 2))
    e = np.full(size.shape, HIGH)
    for up in range(HIGH - 1, LOW - 1, -1):
        e = np.where(TOP * 2.0 ** up >= size, up, e)
    return e


def page_bytes(page, D):
    return page * D + -(-(page // 16) // 32) * 32


class Pool:
    """A cache [pages, Hkv, bytes] in NumPy and what its rows hold."""

    def __init__(self, pages, hkv, page, D, fill=0):
        self.page, self.D, self.hkv = page, D, hkv
        self.bytes = np.full((pages, hkv, page_bytes(page, D)), fill, np.uint8)

    def parts(self):
        """Codes [pages, Hkv, page, D] and exponents' bytes [pages, Hkv, page / 16], as views."""
        at, b = self.page * self.D, self.bytes
        return b[..., :at].reshape(b.shape[:2] + (self.page, self.D)), b[..., at:at + self.page // 16]

    def write(self, slots, x):
        """One call: runs of tokens that go to one block."""
        slots, x = np.asarray(slots, np.int64), np.asarray(x, np.float64)
        codes, powers = self.parts()
        t = 0
        while t < len(slots):
            if not 0 <= slots[t] < self.bytes.shape[0] * self.page:
                t += 1
                continue
            end = t + 1
            while end < len(slots) and slots[end] >= 0 and slots[end] // 16 == slots[t] // 16:
                end += 1
            p, r = divmod(int(slots[t]), self.page)
            j, rows = r // 16, slots[t:end] % 16
            e = exponent(x[t:end])
            if 0 not in rows:
                was = np.clip(powers[p, :, j].astype(int) - BIAS, LOW, HIGH)
                e = np.maximum(e, was)
                block = codes[p, :, 16 * j:16 * j + 16]
                moved = nearest(CODES[block] * 2.0 ** (was - e)[:, None, None])
                block[...] = np.where((e > was)[:, None, None], moved, block)
            powers[p, :, j] = e + BIAS
            for i, row in enumerate(rows):
                codes[p, :, 16 * j + row] = nearest(x[t + i] * 2.0 ** -e[:, None].astype(float))
            t = end

    def rows(self, pages, n):
        """Values [n, Hkv, D] of the first n rows over a list of pages."""
        if n == 0:
            return np.zeros((0, self.hkv, self.D))
        codes, powers = self.parts()
        r = np.arange(n)
        p = np.asarray(pages)[r // self.page]
        r = r % self.page
        return CODES[codes[p, :, r]] * 2.0 ** (np.clip(powers[p, :, r // 16].astype(int) - BIAS, LOW, HIGH))[..., None]

    def exponents(self, pages, n):
        """[n, Hkv]"""
        r = np.arange(n)
        p = np.asarray(pages)[r // self.page] if n else r
        return np.clip(self.parts()[1][p, :, r % self.page // 16].astype(int) - BIAS, LOW, HIGH)
