"""A rotary plan's tables on the GPU: destroyed once no plan is left that uses
them, and made again for the next."""
import gc

import pytest
import torch

from kunlunxin_fft_amd import execute_rotary_plan, native, plan_rotary, rotary
from kunlunxin_fft_amd.runner import release_retired_plans

pytestmark = pytest.mark.gpu


def test_tables_are_destroyed_and_made_again(gpu):
    x = torch.randn(5, 2, 64, device=gpu)
    positions = torch.arange(5, device=gpu)
    kept = plan_rotary(64, base=4321.0)
    want, other = execute_rotary_plan(kept, x, positions), execute_rotary_plan(plan_rotary(64, base=1234.0), x, positions)
    plan_rotary.cache_clear()
    gc.collect()
    release_retired_plans()
    assert native.retired_count() == 0
    assert torch.equal(execute_rotary_plan(kept, x, positions), want)
    assert torch.equal(execute_rotary_plan(plan_rotary(64, base=1234.0), x, positions), other)


def test_plans_that_come_and_go(gpu):
    """A base for every context length: hundreds of plans, each used once."""
    x = torch.randn(3, 1, 32, device=gpu)
    positions = torch.arange(3, device=gpu)
    plan_rotary.cache_clear()
    gc.collect()
    held = len(rotary._NATIVE)  # by others than the cache of plans
    first = execute_rotary_plan(plan_rotary(32, base=5000.0, max_positions=4096), x, positions)
    for i in range(600):
        execute_rotary_plan(plan_rotary(32, base=5000.0 + i, max_positions=4096), x, positions)
    gc.collect()
    assert len(rotary._NATIVE) <= held + 256
    release_retired_plans()  # a process of one Python thread does so by itself, 64 at a time
    assert native.retired_count() == 0
    assert torch.equal(execute_rotary_plan(plan_rotary(32, base=5000.0, max_positions=4096), x, positions), first)
