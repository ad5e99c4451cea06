"""One rotation wherever it is computed: the append's queries, by each of its
kernels, are the rotary plan's, bit for bit (so that a prompt's queries and a
later recomputation of them are the same)."""
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, execute_rotary_plan, plan_rotary
from test_gpu_paged_cache import _i32, _randn, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("dim,rot,layout", [(128, 128, "half"), (128, 128, "interleaved"), (96, 48, "half"), (64, 20, "half"),
                                            (256, 64, "interleaved")])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [70, 0, 33, 200, 1]], ids=["one each", "mixed"])
def test_append_rotates_queries_as_the_plan_does(gpu, counts, dim, rot, layout, dtype):
    plan = plan_rotary(dim, rot_dim=rot, layout=layout)
    starts = [0, 7, 2000, 70000, 5]
    width = -(-max(a + n for a, n in zip(starts, counts)) // 64)
    table, pool = _table([0] * 5, 64, gpu, 1, width=width)  # no pages: keys are skipped
    cache = PagedCache.empty(pool, 2, dim, 64, gpu)
    t = sum(counts)
    q, k = _randn((t, 20, dim), dtype, gpu, 2), _randn((t, 2, dim), dtype, gpu, 3)
    off = None if t == 5 else _i32(lm.offsets_of(counts), gpu)
    got = append_paged_cache(cache, k, k, table, _i32(starts, gpu), offsets=off, rotary=plan, q=q)
    positions = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, counts)]).to(gpu)
    assert torch.equal(got, execute_rotary_plan(plan, q, positions))
