"""Queries whose only token, or only head, has an odd stride that nothing uses."""
import pytest
import torch

from kunlunxin_fft_amd import attend_paged_cache
from test_gpu_paged_cache import _filled, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_strides_of_single_tokens_and_heads(gpu, dtype):
    cache, table = _filled(gpu, [70, 33, 5], 1, 64, 16, dtype, 500)
    one = _randn((2, 135), dtype, gpu, 501)[:, :128].view(2, 2, 64)[:1]  # of a projection 135 wide
    assert one.stride() == (135, 64, 1)
    got = attend_paged_cache(cache, one, table[:1], _i32([70], gpu))
    assert torch.equal(got, attend_paged_cache(cache, one.contiguous(), table[:1], _i32([70], gpu)))
    head = _randn((3 * 64 + 67,), dtype, gpu, 502).as_strided((3, 1, 64), (64, 67, 1))
    got = attend_paged_cache(cache, head, table, _i32([70, 33, 5], gpu))
    assert torch.equal(got, attend_paged_cache(cache, head.contiguous().clone(memory_format=torch.contiguous_format), table, _i32([70, 33, 5], gpu)))
    # where they are used they are refused, as before
    two = _randn((2, 135), dtype, gpu, 503)[:, :128].view(2, 2, 64)
    with pytest.raises(ValueError, match="aligned"):
        attend_paged_cache(cache, two, table[:2], _i32([70, 33], gpu))
