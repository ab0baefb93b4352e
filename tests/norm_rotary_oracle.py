"""Normed heads with rotary positions and their gradients in 64 bits, with bounds for 32-bit arithmetic.

u = 2^-24.  A lane sums up to 16 squares, five exchanges follow, and mean and eps are three roundings more: the argument of the root is
off by 24 u of itself, the root's reciprocal by half of that and two units in the last place, under RHO = 16 u in all.  The rotation's bound is
TURN(t) = 4e-7 + |t| 2^-52 of the pair's two magnitudes (angle, sine and cosine, two products and a sum)."""
import numpy as np

U = 2.0 ** -24
RHO = 16 * U


def angles(pos, freq, axes):
    """[..., R/2] from pos [A, ...]."""
    return np.stack([pos[axes[i] if axes is not None else 0].astype(np.float64) * f for i, f in enumerate(freq)], -1)


def pair(i, half, interleaved):
    return (2 * i, 2 * i + 1) if interleaved else (i, i + half)


def turned(y, t, interleaved, scale, sign, err):
    """y [..., D] by angles t [..., R/2], and what is off in it where y is off by err."""
    half = t.shape[-1]
    z, off = y.copy(), err.copy()
    for i in range(half):
        a, b = pair(i, half, interleaved)
        c, s = np.cos(t[..., i]) * scale, np.sin(t[..., i]) * scale * sign
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        turn = (4e-7 + np.abs(t[..., i]) * 2.0 ** -52) * abs(scale) * (np.abs(y[..., a]) + np.abs(y[..., b]))
        off[..., a] = np.abs(c) * err[..., a] + np.abs(s) * err[..., b] + turn
        off[..., b] = np.abs(c) * err[..., b] + np.abs(s) * err[..., a] + turn
    return z, off


def forward(x, w, t, interleaved=False, scale=1.0, eps=1e-6):
    """x [..., D], w [D] or None, t [..., R/2] broadcastable -> (z, bound)."""
    x = x.astype(np.float64)
    t = np.broadcast_to(t, x.shape[:-1] + t.shape[-1:])
    if w is None:
        return turned(x, t, interleaved, scale, 1.0, np.zeros_like(x))
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = x * r * w
    return turned(y, t, interleaved, scale, 1.0, (RHO + 2 * U) * np.abs(y))


def backward(dz, x, w, t, interleaved=False, scale=1.0, eps=1e-6):
    """-> (dx, its bound, dw, its bound); a lane adds at most every eighth row's part of dw."""
    x, dz = x.astype(np.float64), dz.astype(np.float64)
    t = np.broadcast_to(t, x.shape[:-1] + t.shape[-1:])
    D = x.shape[-1]
    g, eg = turned(dz, t, interleaved, scale, -1.0, np.zeros_like(dz))
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    unit, h = x * r, g * w
    dw = (g * unit).reshape(-1, D).sum(0)
    rows = x.size // D
    edw = (eg * np.abs(unit) + (RHO + 2 * U) * np.abs(g * unit)).reshape(-1, D).sum(0) + (rows / 8 + 64) * U * np.abs(g * unit).reshape(-1, D).sum(0)
    less = (h * x).mean(-1, keepdims=True) * r * r
    eh = np.abs(w) * eg + U * np.abs(h)
    eless = ((eh * np.abs(x)).mean(-1, keepdims=True) + (24 * U + 2 * RHO + 4 * U) * np.abs(h * x).mean(-1, keepdims=True)) * r * r
    dx = r * (h - x * less)
    edx = r * (eh + np.abs(x) * eless + 2 * U * np.abs(x * less)) + (RHO + 2 * U) * r * (np.abs(h) + np.abs(x * less))
    return dx, edx, dw, edw


def within(got, want, bound, eps):
    """Whether got is off by at most the bound and half a step of its type."""
    off = np.abs(got - want)
    room = (bound + eps / 2 * np.abs(want)) * (1 + 1e-6) + 1e-30
    return bool((off <= room).all()), float((off / room).max()) if off.size else 0.0
