"""Rotation with several axes where tokens alone fill the chip and a thread
takes many heads of its token, in fours and a remainder: every load length in
every type, in place in a fused projection, the gradient; and on the way into
the cache, where a token's query heads come in pieces."""
import pytest
import torch

import lm_device_oracle as dev
from kunlunxin_fft_amd import PagedCache, RotaryAxes, append_paged_cache, execute_rotary_plan, plan_rotary
from test_gpu_paged_cache import _i32, _randn, _table

pytestmark = pytest.mark.gpu

CASES = [
    # (batch or None, tokens, heads, dim, rot, layout, pairs, order): loads of 16 bytes
    (None, 8192, 35, 128, 128, "half", (16, 24, 24), "blocks"),
    (2, 4096, 35, 128, 64, "interleaved", (10, 11, 11), "cycle"),
    # shorter ones
    (None, 8191, 35, 64, 20, "half", (3, 3, 4), "cycle"),
    (3, 2731, 35, 64, 20, "interleaved", (1, 9), "blocks"),
    # a few heads a thread: a round of four and the rest, and no whole round
    (None, 2500, 38, 128, 128, "half", (32, 32), "blocks"),
    (None, 1111, 49, 96, 96, "interleaved", (12, 12, 12, 12), "cycle"),
]


def _input(b, t, heads, dim, dtype, gpu, seed, extra=0):
    return _randn((t, heads + extra, dim) if b is None else (b, t, heads + extra, dim), dtype, gpu, seed)


def _places(plan, x, seed):
    return torch.randint(0, 1 << 20, (plan.axes,) + x.shape[:-2], generator=torch.Generator().manual_seed(seed)).to(x.device)


def _check(plan, x, positions, y, inverse=False):
    want, bound = dev.rotate_axes(plan, x, positions, inverse)
    assert bool(((y.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_many_heads(gpu, case, dtype):
    b, t, heads, dim, rot, layout, pairs, order = case
    print("rotary axes, heads", case, dtype, flush=True)
    plan = plan_rotary(dim, rot_dim=rot, layout=layout, axes=RotaryAxes(pairs, order))
    x = _input(b, t, heads, dim, dtype, gpu, 1)
    positions = _places(plan, x, 2)
    for inverse in (False, True):
        y = execute_rotary_plan(plan, x, positions, inverse=inverse)
        _check(plan, x, positions, y, inverse)
        # each head by itself, bit for bit
        for h in range(heads):
            assert torch.equal(execute_rotary_plan(plan, x[..., h:h + 1, :], positions, inverse=inverse), y[..., h:h + 1, :])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", CASES[:4], ids=str)
def test_in_place_in_a_fused_projection(gpu, case, dtype):
    b, t, heads, dim, rot, layout, pairs, order = case
    plan = plan_rotary(dim, rot_dim=rot, layout=layout, axes=RotaryAxes(pairs, order))
    fused = _input(b, t, heads, dim, dtype, gpu, 3, extra=5)
    keep = fused.clone()
    positions = _places(plan, fused, 4)
    want = execute_rotary_plan(plan, keep[..., :heads, :].contiguous(), positions)
    mine = fused[..., :heads, :]
    assert execute_rotary_plan(plan, mine, positions, out=mine) is mine
    assert torch.equal(mine, want) and torch.equal(fused[..., heads:, :], keep[..., heads:, :])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", CASES[:4], ids=str)
def test_gradient(gpu, case, dtype):
    b, t, heads, dim, rot, layout, pairs, order = case
    plan = plan_rotary(dim, rot_dim=rot, layout=layout, axes=RotaryAxes(pairs, order))
    x = _input(b, t, heads, dim, dtype, gpu, 5, extra=2)[..., :heads, :].requires_grad_()
    g = _input(b, t, heads, dim, dtype, gpu, 6)
    positions = _places(plan, x, 7)
    y = execute_rotary_plan(plan, x, positions)
    (got,) = torch.autograd.grad(y, x, g)
    _check(plan, x.detach(), positions, y.detach())
    _check(plan, g, positions, got, inverse=True)


APPEND = [
    # (dim, rot, layout, pairs, query heads, page, counts)
    (128, 128, "half", (16, 24, 24), 30, 64, [2001, 0, 1000]),             # pieces of four heads, the last of two
    (128, 64, "interleaved", (10, 11, 11), 28, 128, [5000, 4501]),         # of sixteen, the last of twelve
    (96, 96, "half", (24, 24), 32, 32, [3000]),
    (64, 32, "interleaved", (4, 4, 4, 4), 33, 16, [7000, 1]),
    (256, 256, "half", (64, 64), 12, 128, [400, 2100]),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, case, dtype):
    """Queries are those that the plan turns alone, bit for bit; codes and
    scales those of the form that takes a pair at a time (of a view whose
    strides allow nothing else)."""
    dim, rot, layout, pairs, hq, page, counts = case
    print("append axes, heads", case, dtype, flush=True)
    heads, t, starts = 2, sum(counts), [7 * i for i in range(len(counts))]
    plan = plan_rotary(dim, rot_dim=rot, layout=layout, axes=RotaryAxes(pairs))
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 8)
    q, k, v = _randn((t, hq + 2 * heads, dim), dtype, gpu, 9).split([hq, heads, heads], 1)
    positions = torch.randint(0, 1 << 20, (plan.axes, t), generator=torch.Generator().manual_seed(10)).to(gpu)
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    made = []
    for odd in (False, True):
        cache = PagedCache.empty(pool, heads, dim, page, gpu)
        if odd:
            spread = torch.zeros((t, heads, dim + 2), dtype=k.dtype, device=gpu)
            spread[..., 1:-1] = k
        got = append_paged_cache(cache, spread[..., 1:-1] if odd else k, v, table, _i32(starts, gpu), offsets=_i32(offsets, gpu),
                                 rotary=plan, positions=positions, q=q)
        assert torch.equal(got, execute_rotary_plan(plan, q, positions))
        made.append(cache)
    for name in ("k", "v"):
        assert torch.equal(*(getattr(c, name).view(torch.uint8) for c in made))
        assert torch.equal(*(getattr(c, name + "_scale") for c in made))
