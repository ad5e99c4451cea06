"""Plain 64-bit forms of the language-model operators, on the CPU."""
import math

import numpy as np
import torch

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# half a unit in the last place, relative; and half the least subnormal step
HALF_ULP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"fp32": 2.0 ** -150, "fp16": 2.0 ** -25, "bf16": 2.0 ** -134}


def pair_index(layout, rot):
    j = np.arange(rot // 2)
    return (j, j + rot // 2) if layout == "half" else (2 * j, 2 * j + 1)


def rotate(x, positions, frequencies, layout, amplitude=1.0, inverse=False):
    """x (..., heads, dim) float64 numpy, positions (...)."""
    a, b = pair_index(layout, 2 * len(frequencies))
    ang = positions.astype(np.float64)[..., None, None] * np.asarray(frequencies)
    z = (x[..., a] + 1j * x[..., b]) * amplitude * np.exp((-1j if inverse else 1j) * ang)
    y = x.copy()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def rotate_bound(x, y, dtype, frequencies, layout, amplitude=1.0):
    """What an element may be off: the root's error (a product of two rounded
    factors, at most 4 * 2^-24 of its size), the two products and their sum in
    32 bits (2 * 2^-24), rounded up to 8 * 2^-24 of |a| + |b|; then one
    rounding to the type."""
    a, b = pair_index(layout, 2 * len(frequencies))
    size = np.zeros_like(x)
    size[..., a] = size[..., b] = abs(amplitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    err = 8 * 2.0 ** -24 * size
    return err + HALF_ULP[dtype] * (np.abs(y) + err) + LEAST[dtype]


def round_code(x):
    """The nearest e4m3 value, ties to even; NaN for what is not finite."""
    with np.errstate(invalid="ignore", over="ignore"):
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
        y = np.round(x / step) * step
    return np.where(np.isfinite(x), y, np.nan)


def block_scale(x):
    """The least 2^e >= 2^-126 with every finite magnitude at most 448 * 2^e."""
    a = np.abs(x[np.isfinite(x)])
    top = a.max() if a.size else 0.0
    if top == 0.0:
        return 2.0 ** -126
    e = math.ceil(math.log2(top / 448.0)) - 2
    while 448.0 * 2.0 ** e < top:
        e += 1
    return 2.0 ** max(e, -126)


class Cache:
    """The cache as float64 codes and scales, filled token by token."""

    def __init__(self, k, v, ks, vs):
        self.k, self.v, self.ks, self.vs = k, v, ks, vs  # codes [pages][heads][size][dim], both

    @classmethod
    def of(cls, cache):
        def np64(t):
            return t.detach().float().cpu().numpy().astype(np.float64)

        v = np64(cache.v)
        p, h, u, d, _ = v.shape
        return cls(np64(cache.k), np.ascontiguousarray(v.transpose(0, 1, 2, 4, 3)).reshape(p, h, u * 16, d),
                   np64(cache.k_scale), np64(cache.v_scale))

    def append(self, k, v, table, starts, counts):
        """k, v float64 (already rotated); the call's tokens of one page count
        for its scale together."""
        size, at = self.k.shape[2], 0
        for b, n in enumerate(counts):
            i = 0
            while i < n:
                pos = starts[b] + i
                o = pos % size
                m = min(size - o, n - i)
                page = table[b][pos // size] if pos // size < len(table[b]) else -1
                if 0 <= page < self.k.shape[0]:
                    for x, codes, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                        for h in range(codes.shape[1]):
                            new = x[at + i:at + i + m, h]
                            s = block_scale(new)
                            if o:
                                old = scale[page, h]
                                s = max(s, old)
                                codes[page, h] = round_code(codes[page, h] * (old / s))
                            scale[page, h] = s
                            codes[page, h, o:o + m] = round_code(new / s)
                i += m
            at += n

    def tokens(self, row, length):
        """K and V (length, heads, dim) of a sequence."""
        size = self.k.shape[2]
        pages = [int(p) for p in row[:-(-length // size)]]
        k = np.concatenate([self.k[p] * self.ks[p][:, None, None] for p in pages], 1)[:, :length]
        v = np.concatenate([self.v[p] * self.vs[p][:, None, None] for p in pages], 1)[:, :length]
        return k.transpose(1, 0, 2), v.transpose(1, 0, 2)


def attend(cache, q, table, lengths, counts, scale, causal=True, window=None, dtype="bf16"):
    """(out, lse, bound) of q float64 (tokens, heads, dim).  The bound: the
    weights rounded to the type (half an ulp of each), scores accumulated in
    32 bits (each within dim * 2^-24 of the sum of magnitudes, twice for the
    maximum), exponentials and sums (2^-18 together), one rounding of the
    output, and the least steps of the type for small weights and values."""
    u, least = HALF_ULP[dtype], LEAST[dtype]
    t, hq, d = q.shape
    out, lse, bound = np.zeros_like(q), np.full((t, hq), -np.inf), np.zeros_like(q)
    group = hq // cache.k.shape[1]
    at = 0
    for b, n in enumerate(counts):
        length = int(lengths[b])
        if n and length > 0:
            k, v = cache.tokens(table[b], length)
            key = np.arange(length)
            for i in range(n):
                pos = length - n + i
                seen = key <= pos if causal else np.ones(length, bool)
                if window:
                    seen &= key > pos - window
                if not seen.any():
                    continue
                for h in range(hq):
                    kk, vv = k[seen, h // group], v[seen, h // group]
                    x = q[at + i, h]
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


def offsets_of(counts):
    c = [0]
    for n in counts:
        c.append(c[-1] + n)
    return c
