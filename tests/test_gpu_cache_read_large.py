"""Cached tokens read back where the outputs are larger than the caches: every
type, ragged starts and lengths, units that begin and end inside, rows of no
sequence, bad pages; bit for bit what indexing gives."""
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import read_paged_cache
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
