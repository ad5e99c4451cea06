"""Query rows of no sequence (before the first offset, past the last): padding of
a batch with a fixed size, as a captured step has it.  They see no key: 0, and
an lse of -infinity."""
import pytest
import torch

from kunlunxin_fft_amd import attend_paged_cache
from test_gpu_paged_cache import _filled, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_length", [None, 64])
@pytest.mark.parametrize("dim,heads,n", [(64, 2, 1), (64, 4, 8), (96, 4, 12), (128, 4, 12), (128, 4, 30), (256, 4, 8)])
@pytest.mark.parametrize("before,after", [(0, 3), (2, 0), (5, 200)])
def test_rows_of_no_sequence(gpu, dim, heads, n, before, after, max_length):
    print("padding", dim, heads, n, before, after, max_length, flush=True)
    lengths = [60, n] if max_length else [2500, n]
    cache, table = _filled(gpu, lengths, 2, dim, 32, "bf16", 600)
    q = _randn((before + 2 * n + after, 2 * heads, dim), "bf16", gpu, 601)
    off = _i32([before, before + n, before + 2 * n], gpu)
    own = q[before:before + 2 * n].contiguous()
    want = attend_paged_cache(cache, own, table, _i32(lengths, gpu), offsets=_i32([0, n, 2 * n], gpu), max_length=max_length)
    # what the output's memory held before
    junk = [torch.full(q.shape, float("nan"), dtype=q.dtype, device=gpu) for _ in range(3)]
    junk += [torch.full(q.shape[:2], float("nan"), device=gpu) for _ in range(3)]
    torch.cuda.synchronize()
    del junk
    out, lse = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, max_length=max_length, return_lse=True)
    rest = torch.ones(q.shape[0], dtype=torch.bool, device=gpu)
    rest[before:before + 2 * n] = False
    assert torch.isfinite(out[~rest]).all() and torch.isfinite(lse[~rest]).all()
    assert ((out[~rest] - want).abs() <= 2.0 ** -6 * (1 + want.abs())).all()  # (another form: rows count for it)
    assert (out[rest] == 0).all() and torch.isneginf(lse[rest]).all()


def test_no_sequence_has_any(gpu):
    cache, table = _filled(gpu, [40, 3], 1, 64, 16, "fp16", 610)
    q = _randn((7, 2, 64), "fp16", gpu, 611)
    for max_length in (None, 40):
        out = attend_paged_cache(cache, q, table, _i32([40, 3], gpu), offsets=_i32([4, 4, 4], gpu), max_length=max_length)
        assert (out == 0).all()
