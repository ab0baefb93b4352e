"""Which axis and which frequency each pair of channels of a rotary position has (plain Python: for torch and NumPy callers)."""
from __future__ import annotations


def rotary_table(rotary_dim, base=10000.0, sections=None, cyclic=False, own_ladder=False):
    """(frequencies, axes, number of axes): two lists of rotary_dim / 2.  `sections`: the pairs of each axis (None: one axis);
    pairs go to the axes section by section, or with `cyclic` in turn, as long as an axis has some left.  Pair i of n turns by
    `base ** (-i / n)` per position; with `own_ladder` each axis counts its own pairs."""
    n = int(rotary_dim) // 2
    sections = [n] if sections is None else [int(s) for s in sections]
    if int(rotary_dim) != 2 * n or n < 1:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if any(s < 0 for s in sections) or sum(sections) != n:
        raise ValueError(f"sections {sections} must add up to rotary_dim / 2 = {n}")
    if not base > 0:
        raise ValueError("base must be positive")
    if cyclic:
        axes = [a for turn in range(max(sections)) for a, s in enumerate(sections) if turn < s]
    else:
        axes = [a for a, s in enumerate(sections) for _ in range(s)]
    seen = [0] * len(sections)
    freq = []
    for i, a in enumerate(axes):
        freq.append(float(base) ** -((seen[a] / sections[a]) if own_ladder else i / n))
        seen[a] += 1
    return freq, axes, len(sections)
