"""Every form of the attention kernel (by the rows a sequence and key head has,
and the head dim), whole and cut over the chip, and NaN values in each."""
import numpy as np
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import attend_paged_cache
from test_gpu_paged_cache import _check, _f64, _filled, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group,n", [(1, 1), (8, 3), (4, 13), (3, 50)])
def test_forms(gpu, dim, group, n, dtype):
    print("form", dim, group, n, dtype, flush=True)
    lengths = [n + 70, n + 33, n]
    cache, table = _filled(gpu, lengths, 2, dim, 32, dtype, 200, size=1.5)
    q = _randn((3 * n, 2 * group, dim), dtype, gpu, 201)
    _check(cache, q, table, lengths, [n] * 3, dtype)
    _check(cache, q, table, lengths, [n] * 3, dtype, window=20)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group,n", [(2, 1), (8, 3), (4, 13), (4, 40)])
def test_forms_cut_over_the_chip(gpu, dim, group, n):
    """A few sequences of thousands of keys: items in many parts, joined."""
    print("cut", dim, group, n, flush=True)
    lengths = [3000, 1500]
    cache, table = _filled(gpu, lengths, 1, dim, 16, "bf16", 210)
    q = _randn((2 * n, group, dim), "bf16", gpu, 211, 2.0)
    _check(cache, q, table, lengths, [n, n], "bf16")


@pytest.mark.parametrize("dim,group,n", [(128, 2, 8), (96, 2, 12), (64, 2, 24), (128, 2, 24), (256, 2, 30), (96, 2, 100)])
def test_nan_values_in_every_form(gpu, dim, group, n):
    """A NaN value of token 80 of 90, channel 37: in the queries that see it, and
    in that channel, alone."""
    length, bad, channel = 90, 80, 37
    cache, table = _filled(gpu, [max(length, n)], 1, dim, 16, "bf16", 220)
    length = max(length, n)
    q = _randn((n, group, dim), "bf16", gpu, 221)
    off = _i32([0, n], gpu)
    clean = lm.Cache.of(cache)
    want, _, bound = lm.attend(clean, _f64(q), table.cpu().numpy(), [length], [n], dim ** -0.5, dtype="bf16")
    cache.v.view(torch.uint8)[int(table[0, bad // 16]), 0, 0, channel, bad % 16] = 0xff
    got = _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=off))
    first = max(0, bad - (length - n))  # the first query that sees it
    assert np.isnan(got[first:, :, channel]).all()
    got[first:, :, channel] = want[first:, :, channel]
    assert (np.abs(got - want) <= bound).all()
