"""Plain 64-bit forms, on the CPU, of rotation with several axes, of cached
tokens read back, and of attention whose first tokens stay visible."""
import numpy as np

import lm_oracle as lm


def rotate_axes(x, positions, plan, inverse=False):
    """x (..., heads, dim) float64 numpy, positions (axes, ...): each pair by its axis."""
    a, b = lm.pair_index(plan.layout, 2 * len(plan.frequencies))
    ang = np.moveaxis(positions[list(plan.axis_of)], 0, -1).astype(np.float64)[..., None, :] * np.asarray(plan.frequencies)
    z = (x[..., a] + 1j * x[..., b]) * plan.amplitude * np.exp((-1j if inverse else 1j) * ang)
    y = x.copy()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def rotate_bound(x, y, dtype, plan):
    return lm.rotate_bound(x, y, dtype, plan.frequencies, plan.layout, plan.amplitude)


def read(cache, table, starts, counts):
    """(k, v) of an ``lm.Cache``: NaN where there is no such token."""
    pages, heads, size, dim = cache.k.shape
    out = np.full((2, sum(counts), heads, dim), np.nan)
    at = 0
    for b, n in enumerate(counts):
        for pos in range(starts[b], starts[b] + n):
            entry = pos // size
            page = table[b][entry] if 0 <= entry < len(table[b]) else -1
            if 0 <= page < pages:
                out[0, at] = cache.k[page, :, pos % size] * cache.ks[page][:, None]
                out[1, at] = cache.v[page, :, pos % size] * cache.vs[page][:, None]
            at += 1
    return out
