"""Rotary positions: pairs of a head's channels turned by their token's position.

Pair ``j`` of ``rot_dim / 2`` of a token at position ``p``, as a complex
value, is multiplied by ``m exp(i p theta_j)``, ``theta_j = base^(-2 j /
rot_dim)``: the same product with unit roots the transforms make, with roots
from two tables made in extended precision on the host.  Channels past
``rot_dim`` are copied.  The gradient is the product with the conjugate roots
(``inverse=True``), which autograd takes by itself.

``plan_rotary`` is host-only, as ``plan_fft`` is; the tables go to a device
with the first execute there.
"""
from __future__ import annotations

import functools
import math
import threading
import weakref
from dataclasses import dataclass

from . import ledger as _ledger
from . import native

MAX_POSITIONS_LIMIT = 1 << 24
MAX_ROT_DIM = 512


@dataclass(frozen=True)
class RotaryScaling:
    """How frequencies change for contexts longer than a model was trained on.

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: the base raised by ``factor^(r / (r - 2))``, which leaves the
      fastest pair alone and divides the slowest by ``factor``;
    * ``"parts"``: pairs that turn at least ``fast`` times over
      ``original_positions`` are left alone, those that turn at most ``slow``
      times are divided by ``factor``, linearly in the number of turns between.

    ``amplitude`` multiplies the rotated channels.
    """

    kind: str
    factor: float
    original_positions: int = 0
    slow: float = 1.0
    fast: float = 32.0
    amplitude: float = 1.0


@dataclass(frozen=True)
class RotaryPlan:
    """A resolved rotation; made by ``plan_rotary``, reused over calls."""

    head_dim: int
    rot_dim: int
    layout: str
    frequencies: tuple
    amplitude: float
    max_positions: int

    def __hash__(self):  # memoised plans: one object per set of arguments
        return id(self)

    def __eq__(self, other):
        return self is other

    def native(self, device_index: int) -> native.NativeRotary:
        """This plan's tables on a device (built on first use, kept while the
        plan is: a HIP graph that uses them needs the plan kept too)."""
        key = (id(self), device_index)
        hit = _NATIVE.get(key)
        if hit is not None and hit[0]() is self:
            return hit[1]
        from .context import device_context
        from .runner import flush_retired_plans

        with _NATIVE_LOCK:
            hit = _NATIVE.get(key)
            if hit is None or hit[0]() is not self:
                flush_retired_plans()
                with device_context(device_index):
                    made = native.NativeRotary(self.frequencies, self.max_positions, self.amplitude, self.layout,
                                               device_index)
                hit = _NATIVE[key] = (weakref.ref(self, lambda _r: _drop(key, _r)), made)
        return hit[1]


# Tables by plan and device: (weak reference to the plan, tables), dropped when
# the plan dies (and destroyed later, see native.release_retired).
_NATIVE: dict = {}
_NATIVE_LOCK = threading.Lock()


def _drop(key, ref) -> None:
    # not under the lock, which the thread that a collection interrupts may hold
    hit = _NATIVE.get(key)
    if hit is not None and hit[0] is ref:
        _NATIVE.pop(key, None)


def _whole(name: str, v) -> int:
    if isinstance(v, bool) or not isinstance(v, int):
        raise TypeError(f"{name} must be an int, got {type(v).__name__}")
    return v


def _number(name: str, v) -> float:
    if isinstance(v, bool) or not isinstance(v, (int, float)):
        raise TypeError(f"{name} must be a number, got {type(v).__name__}")
    if not math.isfinite(v) or v <= 0:
        raise ValueError(f"{name} must be finite and positive, got {v}")
    return float(v)


@functools.lru_cache(maxsize=256, typed=True)
def plan_rotary(head_dim: int, rot_dim: int | None = None, layout: str = "half", base: float = 10000.0,
                scaling: RotaryScaling | None = None, max_positions: int = 1 << 20) -> RotaryPlan:
    """Resolve a rotation (host-only, no torch; the same arguments give the
    same plan).  ``layout`` says which channels form pair ``j``: ``"half"``
    ``(j, j + rot_dim / 2)``, ``"interleaved"`` ``(2 j, 2 j + 1)``."""
    if _whole("head_dim", head_dim) < 2 or head_dim % 2:
        raise ValueError(f"head_dim must be even and at least 2, got {head_dim}")
    r = head_dim if rot_dim is None else _whole("rot_dim", rot_dim)
    if r < 2 or r % 2 or r > min(head_dim, MAX_ROT_DIM):
        raise ValueError(f"rot_dim must be even, in [2, {min(head_dim, MAX_ROT_DIM)}], got {r}")
    if layout not in native.LAYOUT_IDS:
        raise ValueError(f"unknown layout {layout!r}: one of {sorted(native.LAYOUT_IDS)}")
    if not 1 <= _whole("max_positions", max_positions) <= MAX_POSITIONS_LIMIT:
        raise ValueError(f"max_positions must be in [1, {MAX_POSITIONS_LIMIT}], got {max_positions}")
    base = _number("base", base)
    amplitude = 1.0
    if scaling is not None:
        if not isinstance(scaling, RotaryScaling):
            raise TypeError(f"scaling must be a RotaryScaling, got {type(scaling).__name__}")
        factor = _number("scaling.factor", scaling.factor)
        amplitude = _number("scaling.amplitude", scaling.amplitude)
        if scaling.kind == "base":
            if r == 2:
                raise ValueError("scaling kind 'base' needs rot_dim > 2")
            base *= factor ** (r / (r - 2))
    theta = [base ** (-2.0 * j / r) for j in range(r // 2)]
    if scaling is not None and scaling.kind == "linear":
        theta = [t / factor for t in theta]
    elif scaling is not None and scaling.kind == "parts":
        if _whole("scaling.original_positions", scaling.original_positions) < 1:
            raise ValueError("scaling kind 'parts' needs original_positions >= 1")
        slow, fast = _number("scaling.slow", scaling.slow), _number("scaling.fast", scaling.fast)
        if not slow < fast:
            raise ValueError(f"scaling.slow must be less than scaling.fast, got {slow} and {fast}")
        for j, t in enumerate(theta):
            turns = scaling.original_positions * t / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
            theta[j] = t * (keep + (1.0 - keep) / factor)
    elif scaling is not None and scaling.kind != "base":
        raise ValueError(f"unknown scaling kind {scaling.kind!r}: one of ['base', 'linear', 'parts']")
    return RotaryPlan(head_dim, r, layout, tuple(theta), amplitude, max_positions)


# the torch module, the dtype ids, the autograd function and the query for
# forward-mode tangents, once an execute needs them
_torch = None
_DTYPES: dict = {}
_Rotate = None
_has_tangent = None


def _load_torch():
    global _torch, _Rotate, _has_tangent
    import torch

    from . import runner

    native.load()

    def adjacent(t):
        return t.contiguous() if t.stride(-1) != 1 and t.shape[-1] > 1 else t

    class Rotate(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, positions, plan, inverse):
            ctx.save_for_backward(positions)
            ctx.save_for_forward(positions)
            ctx.plan, ctx.inverse = plan, inverse
            return _launch(plan, x, positions, inverse, None)

        @staticmethod
        def backward(ctx, grad):
            # again a Rotate, so that gradients of gradients work
            return Rotate.apply(adjacent(grad), ctx.saved_tensors[0], ctx.plan, not ctx.inverse), None, None, None

        @staticmethod
        def jvp(ctx, tangent, *_):
            return Rotate.apply(adjacent(tangent), ctx.saved_tensors[0], ctx.plan, ctx.inverse)

    _DTYPES.update({torch.float32: native.F32, torch.float16: native.F16, torch.bfloat16: native.BF16})
    _Rotate = Rotate
    _has_tangent = runner.has_tangent
    _torch = torch


def _launch(plan, x, positions, inverse, out):
    from .runner import current_device, stream_handle

    dev = x.get_device()
    if out is None:
        out = _torch.empty(x.shape, dtype=x.dtype, device=x.device)
    xs, os, ps = x.stride(), out.stride(), positions.stride()
    if x.dim() == 3:
        batch, (tokens, heads, dim) = 1, x.shape
        xs, os, ps = (0,) + xs, (0,) + os, (0,) + ps
    else:
        batch, tokens, heads, dim = x.shape
        if positions.dim() == 1:
            ps = (0,) + ps
    args = native.ROTARY_ARGS.pack(
        x.data_ptr(), out.data_ptr(), positions.data_ptr(), xs[0], xs[1], xs[2], os[0], os[1], os[2], ps[0], ps[1],
        batch, tokens, heads, dim, _DTYPES[x.dtype], positions.dtype is _torch.int64,
        native.DIR_IDS["inverse" if inverse else "forward"])
    table = plan.native(dev)
    if current_device() == dev:
        native.rotary_execute(table, args, stream_handle(dev))
    else:
        from .context import device_context

        with device_context(dev):
            native.rotary_execute(table, args, stream_handle(dev))
    return out


def _check(plan, x, positions, out):
    torch = _torch
    if not isinstance(plan, RotaryPlan):
        raise TypeError(f"plan must be a RotaryPlan, got {type(plan).__name__}")
    for name, t in (("x", x), ("positions", positions)) + ((("out", out),) if out is not None else ()):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if x.dim() not in (3, 4):
        raise ValueError(f"x must be (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), got shape "
                         f"{tuple(x.shape)}")
    if x.shape[-1] != plan.head_dim:
        raise ValueError(f"plan expects head_dim {plan.head_dim}, got shape {tuple(x.shape)}")
    lead = tuple(x.shape[:-2])
    if tuple(positions.shape) not in (lead, lead[-1:]):
        raise ValueError(f"positions must have shape {lead}{' or ' + str(lead[-1:]) if len(lead) == 2 else ''}, got "
                         f"{tuple(positions.shape)}")
    if x.stride(-1) != 1:
        raise ValueError("x must have adjacent channels (last stride 1); call .contiguous() first")
    if out is not None:
        if out.dtype != x.dtype:
            raise TypeError(f"out must be {x.dtype}, got {out.dtype}")
        if out.shape != x.shape or out.stride(-1) != 1:
            raise ValueError(f"out must have x's shape {tuple(x.shape)} and adjacent channels")
        if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad) or _has_tangent(x) or _has_tangent(out):
            raise ValueError("out= does not take part in autograd; leave it out, or run under torch.no_grad()")
    if not torch.cuda.is_available():
        raise RuntimeError("no ROCm GPU available; cannot run the rotary kernels")
    for name, t in (("x", x), ("positions", positions)) + ((("out", out),) if out is not None else ()):
        if t.device.type != "cuda" or t.device != x.device:
            raise ValueError(f"{name} must be on the GPU of x, got {t.device}")


def execute_rotary_plan(plan: RotaryPlan, x, positions, *, inverse: bool = False, out=None):
    """Rotate ``x`` ``(tokens, heads, head_dim)`` or ``(batch, tokens, heads,
    head_dim)`` (any strides with adjacent channels; float32, float16 or
    bfloat16, computed in 32 bits) by ``positions`` (``(tokens,)`` or
    ``(batch, tokens)``, int32 or int64) into a new tensor, or into ``out``,
    which may be ``x`` itself.  A position outside ``[0, max_positions)``
    gives NaN.  ``inverse=True`` multiplies by the conjugate roots.  Takes
    part in autograd, reverse and forward mode."""
    if _torch is None:
        _load_torch()
    _check(plan, x, positions, out)
    with _ledger.phase("rotary"):
        if out is None and (x.requires_grad and _torch.is_grad_enabled() or _has_tangent(x)):
            return _Rotate.apply(x, positions, plan, bool(inverse))
        y = _launch(plan, x, positions, bool(inverse), out)
        if out is not None and not out.is_inference():
            # a backward pass that kept `out` must not take the new values for the old
            _torch.autograd.graph.increment_version(out)
        return y
