"""The multi-axis rotation and the rotating paged write in float64 numpy (not a test module)."""

from __future__ import annotations

import numpy as np


def axis_of(sections):
    return np.repeat(np.arange(len(sections)), sections)


def rotate(x, positions, cos, sin, sections, *, inverse=False):
    """x [B, H, S, D], positions [axes, B, S]: (result, bound of its float32
    arithmetic). Each result is two products and a sum: 3 roundings of 2^-24,
    of at most |x1 c| + |x2 s|. A token with a position outside the tables: 0."""
    half = x.shape[-1] // 2
    bad = ((positions < 0) | (positions >= cos.shape[0])).any(0)
    at = np.where(bad[None], 0, positions)[axis_of(sections)].transpose(1, 2, 0)  # [B, S, half]
    i = np.arange(half)
    c1, c2, s1, s2 = (t[at, i + o][:, None] for t in (cos, sin) for o in (0, half))
    x1, x2 = x[..., :half], x[..., half:]
    if inverse:
        s1, s2 = -s2, -s1
    parts = (x1 * c1, -x2 * s1), (x2 * c2, x1 * s2)
    keep = ~bad[:, None, :, None]
    y = np.concatenate([a + b for a, b in parts], -1) * keep
    mag = np.concatenate([np.abs(a) + np.abs(b) for a, b in parts], -1) * keep
    return y, 3 * 2.0 ** -24 * mag


def write(pages, rows, table, own, live):
    """pages with rows [B, H, L, D] written where live [B, L] and the position own [B, L] has a page."""
    pages = pages.copy()
    size = pages.shape[2]
    for b, i in zip(*np.nonzero(live)):
        lp, off = divmod(int(own[b, i]), size)
        if own[b, i] < 0 or lp >= table.shape[1] or not 0 <= table[b, lp] < pages.shape[0]:
            continue
        pages[table[b, lp], :, off] = rows[b, :, i]
    return pages


def tolerance(y, bound, eps):
    """One rounding to a type of step eps (half a step), with its smallest subnormal, on top of `bound`."""
    tiny = 2.0 ** -24 if eps == 2.0 ** -10 else 0.0  # float16: subnormals of 2^-24
    return bound + eps / 2 * (np.abs(y) + bound) + tiny / 2
