"""The oracle by whole matrices is the oracle row by row: outputs, logarithms of
sums and bounds, on the CPU."""
import numpy as np
import pytest
import torch

import lm_device_oracle as dev
import lm_more_oracle as more
import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, RotaryAxes, plan_rotary


def _cache(pages, heads, dim, page, seed):
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randn(shape, generator=g).to(torch.float8_e4m3fn) for shape in ((pages, heads, page, dim), (pages, heads, page // 16, dim, 16))]
    return PagedCache(*codes, *(torch.exp2(torch.randint(-3, 4, (pages, heads), generator=g).float()) for _ in range(2)))


@pytest.mark.parametrize("kw", [{}, {"causal": False}, {"window": 20}, {"window": 20, "sinks": 5}, {"window": 7, "sinks": 40, "causal": False}], ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend(dtype, kw):
    lengths, counts, dim, page = [50, 0, 3, 90], [7, 2, 5, 1], 64, 16
    cache = _cache(12, 2, dim, page, 1)
    table = torch.tensor([[3, 7, 0, 9, -1, -1], [-1] * 6, [5, -1, -1, -1, -1, -1], [11, 1, 2, 4, 6, 8]], dtype=torch.int32)
    q = torch.randn(sum(counts), 6, dim, generator=torch.Generator().manual_seed(2)).to(lm.DTYPES[dtype])
    want = more.attend(lm.Cache.of(cache), q.double().numpy(), table.numpy(), lengths, counts, dim ** -0.5,
                       kw.get("causal", True), kw.get("window"), kw.get("sinks", 0), dtype)
    got = dev.attend(cache, q, table, lengths, counts, **kw)
    for a, b in zip(got[:2], want):
        np.testing.assert_allclose(a.numpy(), b, rtol=1e-12, atol=1e-13)
    seen = np.isfinite(want[1])
    np.testing.assert_allclose(got[2].numpy()[seen], want[2][seen], rtol=1e-9)


@pytest.mark.parametrize("layout,rot", [("half", 32), ("interleaved", 20)])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_rotate_axes(dtype, layout, rot):
    plan = plan_rotary(64, rot_dim=rot, layout=layout, axes=RotaryAxes((rot // 2 - 4, 4), "cycle"))
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 5, 3, 64, generator=g).to(lm.DTYPES[dtype])
    positions = torch.randint(0, 1 << 20, (2, 2, 5), generator=g)
    for inverse in (False, True):
        y, bound = dev.rotate_axes(plan, x, positions, inverse)
        want = more.rotate_axes(x.double().numpy(), positions.numpy(), plan, inverse)
        np.testing.assert_allclose(y.numpy(), want, rtol=1e-12, atol=1e-13)
        np.testing.assert_allclose(bound.numpy(), more.rotate_bound(x.double().numpy(), want, dtype, plan), rtol=1e-9)
