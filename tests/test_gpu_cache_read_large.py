"""Cached tokens read back where the outputs are larger than the caches: every
type, ragged starts and lengths, units that begin and end inside, rows of no
sequence, bad pages; bit for bit what indexing gives.  And the largest and least
of a type."""
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, read_paged_cache
from test_gpu_cache_read import _random
from test_gpu_paged_cache import _i32, _table

pytestmark = pytest.mark.gpu

CASES = [
    # (dim, heads, page, starts, counts, rows before, rows behind)
    (128, 8, 64, [0], [12000], 0, 0),
    (128, 4, 16, [3, 0, 37, 500, 15], [7001, 1, 0, 9000, 4017], 21, 130),
    (96, 5, 48, [47, 5], [11999, 8003], 1, 0),
    (64, 16, 128, [100, 0, 1], [5001, 3333, 4444], 0, 77),
    (256, 2, 32, [31, 16], [6001, 12007], 5, 5),
]


def _indexed(cache, table, starts, counts, before, behind, dtype):
    """Codes times scales by indexing; NaN of what there is not, 0 of no sequence."""
    at = torch.cat([torch.arange(a, a + n, device=table.device) for a, n in zip(starts, counts)])
    seq = torch.arange(len(counts), device=table.device).repeat_interleave(torch.tensor(counts, device=table.device))
    page, slot = table[seq, at // cache.page_size].long(), at % cache.page_size
    bad = (page < 0) | (page >= cache.pages)
    page = page.masked_fill(bad, 0)
    for codes, scale in ((cache.k.view(torch.uint8)[page, :, slot], cache.k_scale),
                         (cache.v.view(torch.uint8)[page, :, slot // 16, :, slot % 16], cache.v_scale)):
        y = codes.contiguous().view(torch.float8_e4m3fn).float() * scale[page][..., None]
        y[bad] = float("nan")
        none = torch.zeros((1,) + tuple(y.shape[1:]), device=y.device)
        yield torch.cat([none.expand(before, -1, -1), y, none.expand(behind, -1, -1)]).to(dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_read(gpu, case, dtype):
    dim, heads, page, starts, counts, before, behind = case
    print("read, large", case, dtype, flush=True)
    dtype = lm.DTYPES[dtype]
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 1)
    cache = _random(gpu, pool, heads, dim, page, 2)
    table[0, 30], table[-1, 7], table[-1, 33] = -1, pool, 1 << 30
    t = before + sum(counts) + behind
    assert 2 * t * heads * dim * dtype.itemsize > 33 << 20
    off = None if len(counts) == 1 else _i32([before + n for n in lm.offsets_of(counts)], gpu)
    got = read_paged_cache(cache, table, _i32(starts, gpu), t, offsets=off, dtype=dtype)
    for y, want in zip(got, _indexed(cache, table, starts, counts, before, behind, dtype)):
        assert bool(want.isnan().any())
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(nan=3.0), want.nan_to_num(nan=3.0))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_the_largest_and_the_least(gpu, dtype):
    """Codes of 256 and more under a scale of 2^120 are past every type; the least
    code is 2^-9, of scales below 2^-124 less than bfloat16's least step, 2^-133,
    and rounded, in float32 (least step 2^-149) exact."""
    scales = [2.0 ** e for e in (120, 119, -123, -124, -125, -126)]
    n = len(scales)
    k = torch.arange(256, dtype=torch.uint8).repeat(n * 16 * 64 // 256).view(n, 1, 16, 64).to(gpu)
    v = k.view(n, 1, 1, 64, 16).clone()
    scale = torch.tensor(scales, device=gpu)[:, None]
    cache = PagedCache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), scale, scale.clone())
    table = torch.arange(n, dtype=torch.int32, device=gpu)[:, None].contiguous()
    got = read_paged_cache(cache, table, _i32([0] * n, gpu), 16 * n, dtype=lm.DTYPES[dtype])
    of = scale.double().repeat_interleave(16, 0)[:, :, None]
    for y, codes in zip(got, (cache.k.view(n * 16, 1, 64), cache.v.view(n, 64, 16).view(torch.uint8).transpose(1, 2).contiguous()
                              .view(torch.float8_e4m3fn).view(n * 16, 1, 64))):
        exact = codes.double() * of
        want = exact.to(lm.DTYPES[dtype])
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(nan=3.0), want.nan_to_num(nan=3.0))
        same = (y.double() == exact) | exact.isnan()
        if dtype == "fp32":
            assert bool(same[16:].all()) and bool(y[:16][codes[:16].double() >= 256].isposinf().all())
        if dtype == "bf16":
            assert bool(same[16:64].all()) and not bool(same[64:].all())
