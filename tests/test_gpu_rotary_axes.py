"""Rotary positions with several axes against the 64-bit form: types, layouts,
orders, ladders, parts of a head, strides of every operand, in place, the
gradient, another stream, a graph; and on the way into the cache."""
import numpy as np
import pytest
import torch

import lm_more_oracle as more
import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, RotaryAxes, RotaryScaling, append_paged_cache, execute_rotary_plan, plan_rotary
from test_gpu_paged_cache import _f64, _i32, _randn, _same, _table
from test_gpu_rotary import _x

pytestmark = pytest.mark.gpu


def _places(plan, shape, gpu, seed, top=1 << 20):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, top, (plan.axes,) + tuple(shape), generator=g).to(gpu)


def _check(plan, x, positions, y, dtype, inverse=False):
    xs = _f64(x)
    pos = positions.cpu().numpy()
    pos = np.broadcast_to(pos if pos.ndim == xs.ndim - 1 else pos[:, None], (plan.axes,) + xs.shape[:-2])
    want = more.rotate_axes(xs, pos, plan, inverse)
    off = np.abs(_f64(y) - want)
    bound = more.rotate_bound(xs, want, dtype, plan)
    assert (off <= bound).all(), f"worst {np.max(off - bound)} past the bound"


CASES = [
    # (batch or None, tokens, heads, dim, rot, layout, pairs, order, ladder)
    (None, 1, 1, 4, 4, "half", (1, 1), "blocks", "own"),
    (None, 1, 40, 128, 128, "half", (16, 24, 24), "blocks", "shared"),
    (None, 33, 3, 128, 128, "interleaved", (16, 24, 24), "cycle", "shared"),
    (None, 257, 5, 96, 48, "half", (3, 4, 5, 12), "cycle", "own"),
    (None, 100, 2, 80, 20, "interleaved", (1, 9), "blocks", "own"),
    (None, 100, 2, 80, 20, "half", (3, 3, 4), "blocks", "shared"),
    (2, 65, 4, 64, 64, "half", (8, 12, 12), "blocks", "shared"),
    (3, 7, 2, 256, 128, "interleaved", (32, 32), "blocks", "own"),
    (2, 513, 7, 18, 6, "half", (1, 1, 1), "cycle", "shared"),
    (4, 1, 64, 512, 512, "half", (64, 64, 64, 64), "cycle", "shared"),
    (1, 1000, 9, 64, 16, "interleaved", (8,), "blocks", "own"),
    (None, 4099, 33, 32, 32, "half", (5, 11), "cycle", "own"),
    (2, 3000, 16, 64, 64, "half", (10, 11, 11), "blocks", "own"),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotation(gpu, case, dtype):
    b, t, h, d, r, layout, pairs, order, ladder = case
    print("rotary axes", case, dtype, flush=True)
    plan = plan_rotary(d, rot_dim=r, layout=layout, axes=RotaryAxes(pairs, order, ladder))
    x = _x(((t, h, d) if b is None else (b, t, h, d)), dtype, gpu, t)
    positions = _places(plan, x.shape[:-2], gpu, t + 1)
    for inverse in (False, True):
        y = execute_rotary_plan(plan, x, positions, inverse=inverse)
        assert y.dtype == x.dtype and y.shape == x.shape
        _check(plan, x, positions, y, dtype, inverse)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_axes_that_agree_are_one_axis(gpu, dtype, layout):
    """Text: the same position along every axis, bit for bit as without axes."""
    x = _x((2, 300, 5, 128), dtype, gpu, 1)
    p = torch.arange(300, device=gpu) + 70000
    want = execute_rotary_plan(plan_rotary(128, layout=layout), x, p)
    for pairs in ((16, 24, 24), (64,), (1, 63)):
        plan = plan_rotary(128, layout=layout, axes=RotaryAxes(pairs))
        assert torch.equal(execute_rotary_plan(plan, x, p.expand(len(pairs), 300)), want)


def test_position_types_and_strides(gpu):
    plan = plan_rotary(64, axes=RotaryAxes((8, 12, 12)))
    x = _x((2, 9, 3, 64), "bf16", gpu, 2)
    p = _places(plan, (2, 9), gpu, 3, 5000)
    want = execute_rotary_plan(plan, x, p)
    spread = torch.zeros(9, 4, 2, 6, dtype=torch.int64, device=gpu)
    spread[:, 1, :, :3] = p.permute(2, 1, 0)
    for q in (p.int(), p.transpose(1, 2).contiguous().transpose(1, 2), spread[:, 1, :, :3].permute(2, 1, 0),
              spread[:, 1, :, :3].int().permute(2, 1, 0)):
        assert torch.equal(execute_rotary_plan(plan, x, q), want)
    both = execute_rotary_plan(plan, x, p[:, 0])  # one sequence's positions for the whole batch
    assert torch.equal(both, execute_rotary_plan(plan, x, p[:, :1].expand(3, 2, 9)))


def test_strides_of_x(gpu):
    """Views of a fused projection, heads before tokens, a broadcast batch, odd offsets."""
    plan = plan_rotary(64, rot_dim=32, axes=RotaryAxes((4, 6, 6)))
    positions = _places(plan, (40,), gpu, 4)
    fused = _x((2, 40, 11, 64), "bf16", gpu, 3)
    for x in (fused[:, :, 2:9], fused.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), fused[:1].expand(5, 40, 11, 64),
              fused.reshape(-1)[8:8 + 40 * 3 * 64].view(1, 40, 3, 64), fused.reshape(-1)[1:1 + 40 * 3 * 64].view(1, 40, 3, 64),
              _x((1, 40, 2, 67), "fp16", gpu, 4)[..., 2:66]):
        y = execute_rotary_plan(plan, x, positions)
        _check(plan, x, positions, y, "bf16" if x.dtype == torch.bfloat16 else "fp16")


def test_in_place_and_out(gpu):
    plan = plan_rotary(128, rot_dim=64, axes=RotaryAxes((16, 16), "cycle"))
    positions = _places(plan, (77,), gpu, 5)
    fused = _x((77, 9, 128), "bf16", gpu, 5)
    keep = fused.clone()
    want = execute_rotary_plan(plan, fused[:, :6], positions)
    got = execute_rotary_plan(plan, fused[:, :6], positions, out=fused[:, :6])
    assert torch.equal(got, want) and torch.equal(fused[:, 6:], keep[:, 6:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_out_of_range_give_nan_in_their_axis(gpu, layout):
    plan = plan_rotary(64, rot_dim=32, layout=layout, max_positions=1500, axes=RotaryAxes((5, 11)))
    x = _x((4, 2, 64), "fp32", gpu, 6)
    y = execute_rotary_plan(plan, x, torch.tensor([[-1, 1499, 3, 2], [0, 1499, 1500, 1 << 40]], device=gpu)).cpu()
    a, b = lm.pair_index(layout, 32)
    first, second = (torch.tensor(np.concatenate([a[s], b[s]])) for s in (slice(0, 5), slice(5, 16)))
    assert torch.isnan(y[0][:, first]).all() and torch.isfinite(y[0][:, second]).all() and torch.isfinite(y[1]).all()
    assert torch.isfinite(y[2:][..., first]).all() and torch.isnan(y[2:][..., second]).all()
    assert torch.equal(y[..., 32:], x.cpu()[..., 32:])


def test_empty(gpu):
    plan = plan_rotary(64, axes=RotaryAxes((16, 16)))
    for shape in ((0, 4, 64), (3, 0, 64), (0, 5, 2, 64), (2, 0, 2, 64)):
        x = torch.zeros(shape, device=gpu, requires_grad=True)
        y = execute_rotary_plan(plan, x, torch.zeros((2,) + shape[:-2], dtype=torch.int64, device=gpu))
        y.sum().backward()
        assert y.shape == x.shape and x.grad.shape == x.shape


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout,order", [("half", "blocks"), ("interleaved", "cycle")])
def test_gradient_is_the_formula(gpu, layout, order, dtype):
    plan = plan_rotary(96, rot_dim=48, layout=layout, scaling=RotaryScaling("linear", 2.0, amplitude=1.25),
                       axes=RotaryAxes((4, 10, 10), order))
    x = _x((2, 31, 3, 96), dtype, gpu, 7).requires_grad_()
    positions = _places(plan, (2, 31), gpu, 8, 3000)
    g = _x((2, 31, 3, 96), dtype, gpu, 8)
    execute_rotary_plan(plan, x, positions).backward(g)
    _check(plan, g, positions, x.grad, dtype, inverse=True)


def test_gradient_against_differences(gpu):
    """The rotation is linear, so a difference over any step is its derivative
    up to the 32-bit rounding of the two values: 8 * 2^-24 of |x| + |d| of a
    pair each, over 2 e = 1, against |g|."""
    plan = plan_rotary(64, rot_dim=40, layout="interleaved", axes=RotaryAxes((6, 7, 7), ladder="own"))
    x, d, g = (_x((17, 5, 64), "fp32", gpu, s) for s in (9, 10, 11))
    positions = _places(plan, (17,), gpu, 12, 5000)
    x.requires_grad_()
    execute_rotary_plan(plan, x, positions).backward(g)
    e = 0.5
    with torch.no_grad():
        diff = (execute_rotary_plan(plan, x + e * d, positions).double()
                - execute_rotary_plan(plan, x - e * d, positions).double()) / (2 * e)
    got = float((x.grad.double() * d.double()).sum())
    want = float((g.double() * diff).sum())
    size = (x.detach().abs() + d.abs()).double().sum(-1, keepdim=True)
    bound = 2.0 ** -20 * float((g.abs().double() * size).sum())
    assert abs(got - want) <= bound


def test_gradient_of_broadcast_heads_and_second_gradient(gpu):
    plan = plan_rotary(64, axes=RotaryAxes((8, 24)))
    positions = _places(plan, (20,), gpu, 13, 900)
    x = _x((20, 1, 64), "fp32", gpu, 12).requires_grad_()
    g = _x((20, 6, 64), "fp32", gpu, 13)
    execute_rotary_plan(plan, x.expand(20, 6, 64), positions).backward(g)
    one = more.rotate_axes(_f64(g), positions.cpu().numpy(), plan, inverse=True).sum(1, keepdims=True)
    tol = 16 * 2.0 ** -24 * (np.abs(_f64(g)).sum(1, keepdims=True).sum(-1, keepdims=True) + 1)
    assert (np.abs(_f64(x.grad) - one) <= tol).all()
    y = _x((20, 2, 64), "fp32", gpu, 14).requires_grad_()
    h = _x((20, 2, 64), "fp32", gpu, 15).requires_grad_()
    (dy,) = torch.autograd.grad(execute_rotary_plan(plan, y, positions), y, h, create_graph=True)
    w = _x((20, 2, 64), "fp32", gpu, 16)
    (dh,) = torch.autograd.grad(dy, h, w)
    _check(plan, w, positions, dh, "fp32")


def test_side_stream_and_graph(gpu):
    plan = plan_rotary(128, axes=RotaryAxes((16, 24, 24)))
    x = _x((300, 8, 128), "bf16", gpu, 17)
    positions = _places(plan, (300,), gpu, 18)
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
        positions.copy_(_places(plan, (300,), gpu, 30 + k))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, execute_rotary_plan(plan, x, positions))
    del graph


APPEND = [
    # (dim, rot, layout, pairs or None, dtype, starts, counts, extra rows before and behind)
    (128, 128, "half", (16, 24, 24), "bf16", [0, 40, 5], [70, 1, 0], 0),
    (128, 64, "interleaved", (8, 24), "fp16", [3, 0], [100, 33], 0),
    (64, 20, "half", (3, 3, 4), "fp32", [0, 17, 31], [1, 1, 1], 0),
    (96, 96, "half", None, "bf16", [10, 0], [50, 20], 3),
    (256, 256, "interleaved", (64, 64), "fp32", [0], [40], 0),
    (64, 64, "half", (8, 8, 8, 8), "bf16", [15, 0, 2], [1, 1, 1], 0),
]


@pytest.mark.parametrize("wide", [False, True], ids=["int32", "int64"])
@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append_turns_by_positions(gpu, case, wide):
    """Keys and queries turned by positions that are not their places."""
    dim, rot, layout, pairs, dtype, starts, counts, extra = case
    print("append axes", case, flush=True)
    heads, hq, page = 2, 6, 32
    plan = plan_rotary(dim, rot_dim=rot, layout=layout, axes=None if pairs is None else RotaryAxes(pairs, "cycle"))
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 6)
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    want = lm.Cache.of(cache)
    t = sum(counts)
    fused = _randn((t + 2 * extra, hq + 2 * heads, dim), dtype, gpu, 7)
    q, k, v = fused.split([hq, heads, heads], 1)
    positions = torch.randint(0, 1 << 19, (max(1, plan.axes), t + 2 * extra), generator=torch.Generator().manual_seed(8))
    pos = positions.numpy()[:, extra:extra + t]
    positions = positions.to(gpu) if wide else positions.int().to(gpu)
    off = _i32([extra + o for o in lm.offsets_of(counts)], gpu)
    if not plan.axes:
        positions = positions[0]
    if all(n == 1 for n in counts) and not extra:
        off = None
    got = append_paged_cache(cache, k, v, table, _i32(starts, gpu), offsets=off, rotary=plan, q=q, positions=positions)
    mine = slice(extra, extra + t)

    def turned(x):
        if plan.axes:
            return more.rotate_axes(_f64(x)[mine], pos, plan)
        return lm.rotate(_f64(x)[mine], pos[0], plan.frequencies, layout)

    want.append(turned(k), _f64(v)[mine], table.cpu().numpy(), starts, counts)
    _same(cache, want, exact_k=False)
    qr = turned(q)
    assert (np.abs(_f64(got)[mine] - qr) <= more.rotate_bound(_f64(q)[mine], qr, dtype, plan)).all()


@pytest.mark.parametrize("axes", [None, RotaryAxes((16, 24, 24))], ids=["one", "three"])
def test_append_by_places_is_append_by_positions_that_are_them(gpu, axes):
    """Bit for bit, whichever call a program makes; and a query turned on the
    way is the one that the plan turns alone."""
    dim, heads, hq, page, starts, counts = 128, 2, 8, 64, [0, 100, 7], [130, 64, 3]
    t = sum(counts)
    fused = _randn((t, hq + 2 * heads, dim), "bf16", gpu, 9)
    q, k, v = fused.split([hq, heads, heads], 1)
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 6)
    places = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, counts)]).to(gpu)
    plain = plan_rotary(dim)
    plan = plan_rotary(dim, axes=axes)
    made = []
    for kw in (dict(rotary=plain), dict(rotary=plan, positions=places.expand(3, t) if axes else places)):
        cache = PagedCache.empty(pool, heads, dim, page, gpu)
        y = append_paged_cache(cache, k, v, table, _i32(starts, gpu), offsets=_i32(lm.offsets_of(counts), gpu), q=q, **kw)
        made.append((cache, y))
    (a, ya), (b, yb) = made
    assert torch.equal(ya, yb) and torch.equal(ya, execute_rotary_plan(plain, q, places))
    for x in ("k", "v"):
        assert torch.equal(getattr(a, x).view(torch.uint8), getattr(b, x).view(torch.uint8))
        assert torch.equal(getattr(a, x + "_scale"), getattr(b, x + "_scale"))


def test_append_positions_out_of_range(gpu):
    """A position that the plan does not hold: NaN codes in the pairs of its
    axis, which do not count for the page's scale; the others as ever."""
    plan = plan_rotary(64, max_positions=100, axes=RotaryAxes((16, 16)))
    cache = PagedCache.empty(1, 1, 64, 16, gpu)
    k = _randn((2, 1, 64), "fp32", gpu, 10)
    positions = _i32([[5, 100], [7, 8]], gpu)
    append_paged_cache(cache, k, k, _i32([[0]], gpu), _i32([0], gpu), offsets=_i32([0, 2], gpu), rotary=plan, positions=positions)
    want = lm.Cache(*(np.zeros((1, 1, 16, 64)) for _ in range(2)), *(np.full((1, 1), 2.0 ** -126) for _ in range(2)))
    turned = more.rotate_axes(_f64(k), np.array([[5, 0], [7, 8]]), plan)
    turned[1, :, list(range(16)) + list(range(32, 48))] = np.nan
    want.append(turned, _f64(k), [[0]], [0], [2])
    got = lm.Cache.of(cache)
    np.testing.assert_array_equal(np.isnan(got.k), np.isnan(want.k))
    got.k[np.isnan(got.k)] = want.k[np.isnan(want.k)] = 0
    assert got.ks == want.ks and (np.abs(got.k - want.k) <= np.maximum(np.abs(want.k) * 2.0 ** -3, 2.0 ** -9)).all()
