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


def attend(cache, q, table, lengths, counts, scale, causal=True, window=None, sinks=0, dtype="bf16"):
    """``lm.attend`` with the first ``sinks`` keys visible beside a window.  The
    same bound: what it counts does not ask which keys are seen."""
    if not (window and sinks):
        return lm.attend(cache, q, table, lengths, counts, scale, causal, window, dtype)
    u, least = lm.HALF_ULP[dtype], lm.LEAST[dtype]
    t, hq, d = q.shape
    out, lse, bound = np.zeros_like(q), np.full((t, hq), -np.inf), np.zeros_like(q)
    group, at = hq // cache.k.shape[1], 0
    for b, n in enumerate(counts):
        length = int(lengths[b])
        if n and length > 0:
            k, v = tokens(cache, table[b], length)
            key = np.arange(length)
            for i in range(n):
                pos = length - n + i
                seen = (key <= pos if causal else np.ones(length, bool)) & ((key > pos - window) | (key < sinks))
                if not seen.any():
                    continue
                for h in range(hq):
                    kk, vv, x = k[seen, h // group], v[seen, h // group], q[at + i, h]
                    s = (kk @ x) * scale
                    size = scale * (np.abs(kk) @ np.abs(x)).max()
                    m = s.max()
                    p = np.exp(s - m)
                    total = p.sum()
                    out[at + i, h] = (p / total) @ vv
                    lse[at + i, h] = m + np.log(total)
                    weight = (p / total) @ np.abs(vv)
                    off = weight * (u + 2.0 ** -18 + 2 * d * 2.0 ** -24 * size)
                    off += len(p) * least * np.abs(vv).max() / total + least
                    bound[at + i, h] = off + u * (np.abs(out[at + i, h]) + off) + least
        at += n
    return out, lse, bound


def tokens(cache, row, length):
    """K and V (length, heads, dim) of a sequence; NaN of pages that are none."""
    pages, _, size, _ = cache.k.shape
    k, v = (np.concatenate([(x[p] * s[p][:, None, None]) if 0 <= p < pages else np.full(x[0].shape, np.nan)
                            for p in map(int, row[:-(-length // size)])], 1)[:, :length] for x, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
    return k.transpose(1, 0, 2), v.transpose(1, 0, 2)
