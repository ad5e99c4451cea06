"""Rotary positions against the 64-bit form: types, layouts, parts of a head,
long positions, strides, in place, the gradient, other streams, graphs."""
import math

import numpy as np
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import RotaryScaling, execute_rotary_plan, plan_rotary

pytestmark = pytest.mark.gpu


def _x(shape, dtype, gpu, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * 3).to(lm.DTYPES[dtype]).to(gpu)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _check(plan, x, positions, y, dtype, inverse=False):
    xs = _f64(x)
    pos = np.broadcast_to(positions.cpu().numpy(), xs.shape[:-2])
    want = lm.rotate(xs, pos, plan.frequencies, plan.layout, plan.amplitude, inverse)
    bound = lm.rotate_bound(xs, want, dtype, plan.frequencies, plan.layout, plan.amplitude)
    off = np.abs(_f64(y) - want)
    assert (off <= bound).all(), f"worst {np.max(off - bound)} past the bound"


CASES = [
    # (batch or None, tokens, heads, dim, rot, layout)
    (None, 1, 1, 2, 2, "half"),
    (None, 1, 40, 128, 128, "half"),
    (None, 33, 3, 128, 128, "interleaved"),
    (None, 257, 5, 96, 48, "half"),
    (None, 100, 2, 80, 20, "interleaved"),
    (None, 100, 2, 80, 20, "half"),
    (2, 65, 4, 64, 64, "half"),
    (3, 7, 2, 256, 128, "interleaved"),
    (2, 513, 7, 18, 6, "half"),
    (4, 1, 64, 512, 512, "half"),
    (1, 1000, 9, 64, 16, "interleaved"),
    (None, 4099, 33, 32, 32, "half"),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotation(gpu, case, dtype):
    b, t, h, d, r, layout = case
    print("rotary", case, dtype, flush=True)
    plan = plan_rotary(d, rot_dim=r, layout=layout)
    x = _x(((t, h, d) if b is None else (b, t, h, d)), dtype, gpu, t)
    g = torch.Generator().manual_seed(t + 1)
    positions = torch.randint(0, 1 << 20, x.shape[:-2], generator=g).to(gpu)
    for inverse in (False, True):
        y = execute_rotary_plan(plan, x, positions, inverse=inverse)
        assert y.dtype == x.dtype and y.shape == x.shape
        _check(plan, x, positions, y, dtype, inverse)


@pytest.mark.parametrize("scaling", [
    RotaryScaling("linear", 8.0), RotaryScaling("base", 4.0, amplitude=1.2),
    RotaryScaling("parts", 16.0, 4096, 1.0, 32.0, 0.1 * math.log(16.0) + 1.0)], ids=lambda s: s.kind)
def test_scaled_frequencies_at_long_positions(gpu, scaling):
    """Every frequency against its formula, and the last positions the plan holds."""
    r, top = 64, 1 << 22
    plan = plan_rotary(64, scaling=scaling, max_positions=top, base=500000.0)
    j = np.arange(r // 2)
    theta = 500000.0 ** (-2.0 * j / r)
    if scaling.kind == "linear":
        theta = theta / 8
    elif scaling.kind == "base":
        theta = (500000.0 * 4.0 ** (r / (r - 2))) ** (-2.0 * j / r)
    else:
        keep = np.clip((4096 * theta / (2 * np.pi) - 1) / 31, 0, 1)
        theta = theta * keep + theta / 16 * (1 - keep)
    np.testing.assert_allclose(plan.frequencies, theta, rtol=1e-12)
    x = _x((5, 3, 64), "fp32", gpu, 1)
    positions = torch.tensor([0, 1023, 1024, top - 1025, top - 1], dtype=torch.int32, device=gpu)
    _check(plan, x, positions, execute_rotary_plan(plan, x, positions), "fp32")


def test_position_types_and_shapes(gpu):
    plan = plan_rotary(64)
    x = _x((2, 9, 3, 64), "bf16", gpu, 2)
    p64 = torch.arange(9, device=gpu) * 11
    want = execute_rotary_plan(plan, x, p64.expand(2, 9).contiguous())
    for p in (p64, p64.int(), p64.expand(2, 9), p64.int().expand(2, 9).contiguous()):
        assert torch.equal(execute_rotary_plan(plan, x, p), want)
    strided = torch.stack([p64, p64 + 1], 1)[:, 0]
    assert torch.equal(execute_rotary_plan(plan, x, strided), want)


def test_strides(gpu):
    """Views of a fused projection, heads before tokens, a broadcast batch, odd offsets."""
    plan = plan_rotary(64, rot_dim=32)
    positions = torch.arange(50, 90, device=gpu)
    fused = _x((2, 40, 11, 64), "bf16", gpu, 3)
    for x in (fused[:, :, 2:9], fused.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), fused[:1].expand(5, 40, 11, 64),
              fused.reshape(-1)[8:8 + 40 * 3 * 64].view(1, 40, 3, 64), fused.reshape(-1)[1:1 + 40 * 3 * 64].view(1, 40, 3, 64),
              _x((1, 40, 2, 67), "fp16", gpu, 4)[..., 2:66]):
        y = execute_rotary_plan(plan, x, positions)
        _check(plan, x, positions, y, "bf16" if x.dtype == torch.bfloat16 else "fp16")


def test_in_place_and_out(gpu):
    plan = plan_rotary(128, rot_dim=64)
    positions = torch.arange(77, device=gpu)
    fused = _x((77, 9, 128), "bf16", gpu, 5)
    keep = fused.clone()
    want = execute_rotary_plan(plan, fused[:, :6], positions)
    got = execute_rotary_plan(plan, fused[:, :6], positions, out=fused[:, :6])
    assert torch.equal(got, want) and torch.equal(fused[:, 6:], keep[:, 6:])
    out = torch.full((77, 12, 128), 7.0, dtype=torch.bfloat16, device=gpu)
    execute_rotary_plan(plan, keep[:, :6], positions, out=out[:, 3:9])
    assert torch.equal(out[:, 3:9], want)
    assert bool((out[:, :3] == 7).all()) and bool((out[:, 9:] == 7).all())


def test_positions_out_of_range_give_nan(gpu):
    plan = plan_rotary(64, rot_dim=32, max_positions=1500)
    x = _x((4, 2, 64), "fp32", gpu, 6)
    y = execute_rotary_plan(plan, x, torch.tensor([-1, 1499, 1500, 1 << 40], device=gpu)).cpu()
    assert torch.isfinite(y[1]).all() and torch.isnan(y[[0, 2, 3], :, :32]).all()
    assert torch.equal(y[..., 32:], x.cpu()[..., 32:])  # copied whatever the position


def test_empty(gpu):
    plan = plan_rotary(64)
    for shape in ((0, 4, 64), (3, 0, 64), (0, 5, 2, 64), (2, 0, 2, 64)):
        x = torch.zeros(shape, device=gpu, requires_grad=True)
        y = execute_rotary_plan(plan, x, torch.zeros(shape[:-2], dtype=torch.int64, device=gpu))
        y.sum().backward()
        assert y.shape == x.shape and x.grad.shape == x.shape


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_formula(gpu, layout, dtype):
    plan = plan_rotary(96, rot_dim=48, layout=layout, scaling=RotaryScaling("linear", 2.0, amplitude=1.25))
    x = _x((2, 31, 3, 96), dtype, gpu, 7).requires_grad_()
    positions = torch.arange(31, device=gpu)
    g = _x((2, 31, 3, 96), dtype, gpu, 8)
    execute_rotary_plan(plan, x, positions).backward(g)
    _check(plan, g, positions, x.grad, dtype, inverse=True)


def test_gradient_against_differences(gpu):
    """<g, (f(x + e d) - f(x - e d)) / 2 e> = <df/dx^T g, d>: f is linear, so
    the difference is exact up to the 32-bit rounding of f, 2^-22 of |f| / e."""
    plan = plan_rotary(64, rot_dim=40, layout="interleaved")
    x, d, g = (_x((17, 5, 64), "fp32", gpu, s) for s in (9, 10, 11))
    positions = torch.arange(1000, 1017, device=gpu)
    x.requires_grad_()
    execute_rotary_plan(plan, x, positions).backward(g)
    e = 0.5
    with torch.no_grad():
        diff = (execute_rotary_plan(plan, x + e * d, positions).double()
                - execute_rotary_plan(plan, x - e * d, positions).double()) / (2 * e)
    got = float((x.grad.double() * d.double()).sum())
    want = float((g.double() * diff).sum())
    bound = 2.0 ** -20 * float((g.abs() * (x.abs() + d.abs()).sum(-1, keepdim=True)).sum())
    assert abs(got - want) <= bound


def test_gradient_of_broadcast_and_shared_heads(gpu):
    """One key head rotated for several query heads, and a broadcast gradient
    (stride 0 in every dimension, as .sum() sends back)."""
    plan = plan_rotary(64)
    positions = torch.arange(20, device=gpu)
    x = _x((20, 1, 64), "fp32", gpu, 12).requires_grad_()
    g = _x((20, 6, 64), "fp32", gpu, 13)
    execute_rotary_plan(plan, x.expand(20, 6, 64), positions).backward(g)
    one = lm.rotate(_f64(g), np.arange(20), plan.frequencies, "half", inverse=True).sum(1, keepdims=True)
    # six products within 8 * 2^-24 of their pairs, and their 32-bit sum
    tol = 16 * 2.0 ** -24 * (np.abs(_f64(g)).sum() + 1)
    assert np.abs(_f64(x.grad) - one).max() <= tol
    x.grad = None
    execute_rotary_plan(plan, x, positions).sum().backward()
    want = lm.rotate(np.ones((20, 1, 64)), np.arange(20), plan.frequencies, "half", inverse=True)
    assert np.abs(_f64(x.grad) - want).max() <= 16 * 2.0 ** -24 * 2


def test_second_gradient(gpu):
    plan = plan_rotary(64)
    positions = torch.arange(8, device=gpu)
    x = _x((8, 2, 64), "fp32", gpu, 14).requires_grad_()
    g = _x((8, 2, 64), "fp32", gpu, 15).requires_grad_()
    (dx,) = torch.autograd.grad(execute_rotary_plan(plan, x, positions), x, g, create_graph=True)
    w = _x((8, 2, 64), "fp32", gpu, 16)
    (dg,) = torch.autograd.grad(dx, g, w)
    _check(plan, w, positions, dg, "fp32")


def test_side_stream_and_graph(gpu):
    plan = plan_rotary(128)
    x = _x((300, 8, 128), "bf16", gpu, 17)
    positions = torch.arange(300, device=gpu)
    want = execute_rotary_plan(plan, x, positions)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        assert torch.equal(execute_rotary_plan(plan, x, positions), want)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = execute_rotary_plan(plan, x, positions)
    torch.cuda.synchronize()
    for k in range(3):
        x.copy_(_x((300, 8, 128), "bf16", gpu, 20 + k))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, execute_rotary_plan(plan, x, positions))
    del graph
