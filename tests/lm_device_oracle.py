"""The 64-bit forms of ``lm_oracle`` and ``lm_more_oracle`` by whole matrices on
the tensors' own device, for calls of sizes that those take minutes for: the
same formulas and the same bounds."""
import torch

import lm_oracle as lm

NAMES = {dt: name for name, dt in lm.DTYPES.items()}


def rotate_axes(plan, x, positions, inverse=False):
    """(y, bound) of x (..., heads, dim) turned by positions (axes, ...)."""
    a, b = (torch.from_numpy(i).to(x.device) for i in lm.pair_index(plan.layout, 2 * len(plan.frequencies)))
    theta = torch.tensor(plan.frequencies, dtype=torch.float64, device=x.device)
    angle = positions[list(plan.axis_of)].movedim(0, -1).double()[..., None, :] * theta * (-1 if inverse else 1)
    dtype, x = NAMES[x.dtype], x.double()
    y, size = x.clone(), torch.zeros_like(x)
    cos, sin = plan.amplitude * angle.cos(), plan.amplitude * angle.sin()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = abs(plan.amplitude) * (x[..., a].abs() + x[..., b].abs())
    err = 8 * 2.0 ** -24 * size
    return y, err + lm.HALF_ULP[dtype] * (y.abs() + err) + lm.LEAST[dtype]


def tokens(cache, row, length):
    """K and V (length, heads, dim) of the sequence whose pages ``row`` names."""
    pages = row[:-(-length // cache.page_size)].long()
    k = cache.k[pages].double() * cache.k_scale[pages][..., None, None]
    v = cache.v[pages].double() * cache.v_scale[pages][..., None, None, None]
    return (k.transpose(1, 2).reshape(-1, cache.kv_heads, cache.head_dim)[:length],
            v.permute(0, 2, 4, 1, 3).reshape(-1, cache.kv_heads, cache.head_dim)[:length])


def attend(cache, q, table, lengths, counts, scale=None, causal=True, window=None, sinks=0):
    """(out, lse, bound) of every row, as ``lm.attend``."""
    dtype = NAMES[q.dtype]
    u, least = lm.HALF_ULP[dtype], lm.LEAST[dtype]
    t, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    q = q.double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((t, hq), -torch.inf, dtype=torch.float64, device=q.device)
    group, at = hq // cache.kv_heads, 0
    for b, n in enumerate(counts):
        length = int(lengths[b])
        if n and length > 0:
            k, v = tokens(cache, table[b], length)
            key = torch.arange(length, device=q.device)
            pos = torch.arange(length - n, length, device=q.device)[:, None]
            hidden = (key > pos) if causal else torch.zeros(n, length, dtype=torch.bool, device=q.device)
            if window:
                hidden = hidden | ((key <= pos - window) & (key >= sinks))
            some = ~hidden.all(1)
            rows = slice(at, at + n)
            for h in range(hq):
                kk, vv, x = k[:, h // group].contiguous(), v[:, h // group].contiguous(), q[rows, h].contiguous()
                s = ((x @ kk.T.contiguous()) * scale).masked_fill(hidden, -torch.inf)
                size = scale * (x.abs() @ kk.abs().T.contiguous()).masked_fill(hidden, 0).amax(1, keepdim=True)
                m = s.amax(1, keepdim=True).masked_fill(~some[:, None], 0)
                p = (s - m).exp()
                total = p.sum(1, keepdim=True).masked_fill(~some[:, None], 1)
                y = (p / total) @ vv
                off = ((p / total) @ vv.abs()) * (u + 2.0 ** -18 + 2 * d * 2.0 ** -24 * size)
                large = vv.abs().amax(1).expand(n, length).masked_fill(hidden, 0).amax(1, keepdim=True)
                off = off + (~hidden).sum(1, keepdim=True) * least * large / total + least
                out[rows, h], bound[rows, h] = y, off + u * (y.abs() + off) + least
                lse[rows, h] = (m + total.log()).masked_fill(~some[:, None], -torch.inf)[:, 0]
        at += n
    return out, lse, bound


def check_attend(got, got_lse, want):
    """The worst element against its bound, and the logarithms of sums."""
    out, lse, bound = want
    off = (got.double() - out).abs()
    assert bool((off <= bound).all()), f"worst {float((off / bound).nan_to_num(nan=9e9).max())} of the bound, {int(got.isnan().sum())} NaN"
    empty = lse == -torch.inf
    assert torch.equal(got_lse == -torch.inf, empty) and bool((got[empty] == 0).all())
    assert bool(((got_lse.double() - lse).abs()[~empty] <= 2.0 ** -16 * (1 + lse[~empty].abs())).all())
