"""Attention over values, weights, scores and page scales of any size, in every
form of the kernel (by the rows a sequence and key head has, and the head dim),
whole and cut over the chip."""
import numpy as np
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, attend_paged_cache
from test_gpu_paged_cache import _f64, _i32, _randn

pytestmark = pytest.mark.gpu

# (head dim, query heads, queries): 2, 32, 48, 120 rows to head dim 96; 48 and
# 120 rows of 128; 2 and 32 rows of 256
FORMS = [(64, 2, 1), (64, 4, 8), (96, 4, 12), (96, 4, 30), (128, 4, 12), (128, 4, 30), (256, 2, 1), (256, 4, 8)]


def _cache(gpu, k, v, page, spare=1):
    """A cache of one sequence's k and v (tokens, 1, dim) float32, page 0 and
    `spare - 1` others not its; (cache, table)."""
    n, _, dim = k.shape
    need = -(-n // page)
    cache = PagedCache.empty(need + spare, 1, dim, page, gpu)
    table = torch.arange(spare, need + spare, dtype=torch.int32, device=gpu)[None]
    append_paged_cache(cache, k, v, table, _i32([0], gpu), offsets=_i32([0, n], gpu))
    return cache, table


@pytest.mark.parametrize("length", [150, 3000])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,query", [("bf16", 1e33), ("fp16", 6e4)])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_scores_of_any_size(gpu, dim, heads, n, dtype, query, sign, length):
    """Scores of 2^30 and more, all of one sign: the softmax is the value of the
    largest, alone.  (The weight's own rounding, 2^-11 in float16, is in the
    product and not in the sum.)"""
    print("scores", dim, heads, n, dtype, sign, length, flush=True)
    at = torch.arange(length, device=gpu)
    k = torch.zeros(length, 1, dim, device=gpu)
    size = 1.0 if dtype == "bf16" else 1e6
    k[:, 0, 0] = size * torch.where(at == 5, 1.0 if sign < 0 else 4.0, 2.0 + (at % 3) * 0.25)
    v = _randn((length, 1, dim), "fp32", gpu, 320)
    cache, table = _cache(gpu, k, v, 16)
    q = torch.zeros(n, heads, dim, device=gpu, dtype=lm.DTYPES[dtype])
    q[..., 0] = sign * query
    out, lse = attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu), return_lse=True)
    c = lm.Cache.of(cache)
    ks, vs = c.tokens(table.cpu().numpy()[0], length)
    s = ks[:, 0, 0] * float(q[0, 0, 0]) * dim ** -0.5
    assert s.argmax() == 5 and abs(s[5]) >= 2.0 ** 30
    want = vs[5, 0]
    u = 2.0 ** -11 if dtype == "fp16" else 0.0
    assert (np.abs(_f64(out) - want) <= (u + lm.HALF_ULP[dtype] + 2.0 ** -20) * np.abs(want) + lm.LEAST[dtype]).all()
    assert (np.abs(_f64(lse) - s[5]) <= 2.0 ** -16 * abs(s[5])).all()
