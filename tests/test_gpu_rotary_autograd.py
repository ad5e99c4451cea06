"""Forward-mode differentiation of the rotation, alone and over reverse mode."""
import pytest
import torch
from torch.autograd import forward_ad

from kunlunxin_fft_amd import execute_rotary_plan, plan_rotary
from test_gpu_rotary import _check, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("layout,dtype", [("half", "fp32"), ("interleaved", "bf16")])
def test_tangent_is_rotated(gpu, layout, dtype, inverse):
    plan = plan_rotary(96, rot_dim=48, layout=layout)
    x, t = (_x((2, 31, 3, 96), dtype, gpu, s) for s in (30, 31))
    positions = torch.arange(31, device=gpu)
    with forward_ad.dual_level():
        y = execute_rotary_plan(plan, forward_ad.make_dual(x, t), positions, inverse=inverse)
        value, tangent = forward_ad.unpack_dual(y)
        assert tangent is not None
        _check(plan, x, positions, value, dtype, inverse)
        _check(plan, t, positions, tangent, dtype, inverse)


def test_tangent_of_any_strides(gpu):
    """A tangent with channels that are not adjacent, and one for all heads."""
    plan = plan_rotary(64)
    x = _x((20, 4, 64), "fp32", gpu, 32)
    positions = torch.arange(20, device=gpu)
    for t in (_x((20, 64, 4), "fp32", gpu, 33).transpose(1, 2), _x((20, 1, 64), "fp32", gpu, 34).expand(20, 4, 64)):
        with forward_ad.dual_level():
            y = execute_rotary_plan(plan, forward_ad.make_dual(x, t), positions)
            _check(plan, t, positions, forward_ad.unpack_dual(y).tangent, "fp32")


def test_tangent_of_a_gradient(gpu):
    """Forward over reverse: the gradient's derivative along a tangent of the
    gradient that comes in."""
    plan = plan_rotary(64)
    x = _x((8, 2, 64), "fp32", gpu, 35).requires_grad_()
    g, t = (_x((8, 2, 64), "fp32", gpu, s) for s in (36, 37))
    positions = torch.arange(8, device=gpu)
    with forward_ad.dual_level():
        (dx,) = torch.autograd.grad(execute_rotary_plan(plan, x, positions), x, forward_ad.make_dual(g, t), create_graph=True)
        value, tangent = forward_ad.unpack_dual(dx)
        _check(plan, g, positions, value, "fp32", inverse=True)
        _check(plan, t, positions, tangent, "fp32", inverse=True)


def test_out_refuses_a_tangent(gpu):
    plan = plan_rotary(64)
    x = _x((8, 2, 64), "fp32", gpu, 38)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="autograd"):
            execute_rotary_plan(plan, dual, torch.arange(8, device=gpu), out=torch.empty_like(x))


def test_writing_into_a_saved_tensor_is_noticed(gpu):
    """A tensor another operation keeps for its backward pass, rotated in place,
    or written as out: that backward would be wrong, and says so as it does for
    torch's own in-place operations."""
    plan = plan_rotary(64)
    positions = torch.arange(8, device=gpu)
    for source in ("itself", "another"):
        x = _x((8, 2, 64), "fp32", gpu, 39)
        w = _x((64,), "fp32", gpu, 40).requires_grad_()
        loss = (x * w).sum()
        execute_rotary_plan(plan, x if source == "itself" else x.clone(), positions, out=x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_out_in_inference_mode(gpu):
    plan = plan_rotary(64)
    positions = torch.arange(8, device=gpu)
    x = _x((8, 2, 64), "fp32", gpu, 41)
    want = execute_rotary_plan(plan, x, positions)
    with torch.inference_mode():
        y = x.clone()
        assert execute_rotary_plan(plan, y, positions, out=y) is y
    assert torch.equal(y, want)
