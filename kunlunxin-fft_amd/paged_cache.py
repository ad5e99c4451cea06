"""A paged 8-bit cache of keys and values, the append that fills it and the
attention that reads it.

Codes are e4m3; each page and head shares a power-of-two scale for its keys
and one for its values, the least with every magnitude at most 448 of it:

    k        (pages, kv_heads, page_size, head_dim)            float8_e4m3fn
    v        (pages, kv_heads, page_size / 16, head_dim, 16)   float8_e4m3fn
    k_scale  (pages, kv_heads)                                 float32
    v_scale  (pages, kv_heads)                                 float32

(values lie sixteen tokens of one channel side by side, which is what one lane
of a matrix instruction takes).  Which pages hold a sequence, in order, is the
caller's page table; the library keeps nothing between calls.
"""
from __future__ import annotations

import math

import torch

from . import ledger as _ledger
from . import native
from .context import device_context, device_ready
from .rotary import RotaryPlan
from .runner import current_device, has_tangent, stream_handle

HEAD_DIMS = (64, 96, 128, 256)
MAX_PAGE_SIZE = 1024
# positions of a sequence's table, and of a window
_MAX_POSITIONS = 1 << 30
_DTYPES = {torch.float32: native.F32, torch.float16: native.F16, torch.bfloat16: native.BF16}
# scale of a page nothing was written to: the least there is, so that the
# first tokens decide
_LEAST_SCALE = 2.0 ** -126


def _tensor(name, t, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


class PagedCache:
    """The four tensors of a cache, checked once (layout above), and fixed: the
    kernels use the addresses taken then.  Their contents may be written."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page_size", "head_dim", "device", "_packed")

    def __init__(self, k, v, k_scale, v_scale):
        for name, t, dt in (("k", k, torch.float8_e4m3fn), ("v", v, torch.float8_e4m3fn),
                            ("k_scale", k_scale, torch.float32), ("v_scale", v_scale, torch.float32)):
            _tensor(name, t, dt)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if t.device != k.device:
                raise ValueError(f"{name} must be on {k.device} like k, got {t.device}")
        if k.dim() != 4:
            raise ValueError(f"k must be (pages, kv_heads, page_size, head_dim), got shape {tuple(k.shape)}")
        pages, heads, size, dim = k.shape
        if min(pages, heads) < 1:
            raise ValueError(f"a cache has at least one page and one head, got shape {tuple(k.shape)}")
        if size < 16 or size % 16 or size > MAX_PAGE_SIZE:
            raise ValueError(f"page_size must be a multiple of 16 in [16, {MAX_PAGE_SIZE}], got {size}")
        if dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {dim}")
        if tuple(v.shape) != (pages, heads, size // 16, dim, 16):
            raise ValueError(f"v must have shape {(pages, heads, size // 16, dim, 16)}, got {tuple(v.shape)}")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if tuple(t.shape) != (pages, heads):
                raise ValueError(f"{name} must have shape {(pages, heads)}, got {tuple(t.shape)}")
        packed = native.CACHE_ARGS.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                        pages, heads, dim, size)
        for name, value in zip(self.__slots__, (k, v, k_scale, v_scale, pages, heads, size, dim, k.device, packed)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"a PagedCache's {name} cannot be replaced: make another PagedCache of the tensors")

    def __delattr__(self, name):
        raise AttributeError(f"a PagedCache's {name} cannot be deleted")

    def __reduce__(self):  # a copy takes the addresses of its own tensors
        return PagedCache, (self.k, self.v, self.k_scale, self.v_scale)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> "PagedCache":
        """A cache of ``pages`` pages nothing was written to."""
        if not isinstance(page_size, int) or page_size % 16 or page_size < 16:
            raise ValueError(f"page_size must be a multiple of 16 in [16, {MAX_PAGE_SIZE}], got {page_size}")
        shape = (pages, kv_heads)
        k = torch.zeros(shape + (page_size, head_dim), dtype=torch.uint8, device=device)
        v = torch.zeros(shape + (page_size // 16, head_dim, 16), dtype=torch.uint8, device=device)
        return cls(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn),
                   torch.full(shape, _LEAST_SCALE, device=device), torch.full(shape, _LEAST_SCALE, device=device))


def _index(name, t, device, dim):
    _tensor(name, t, torch.int32)
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimension{'s' if dim > 1 else ''}, got shape {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device} like the cache, got {t.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have adjacent entries (last stride 1); call .contiguous() first")


def _heads(name, t, cache, dtype=None, heads=None):
    _tensor(name, t, dtype)
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.dim() != 3 or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be (tokens, {heads if heads is not None else 'heads'}, {cache.head_dim}), got "
                         f"shape {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have adjacent channels (last stride 1); call .contiguous() first")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on {cache.device} like the cache, got {t.device}")


def _sequences(cache, page_table, lengths, what, offsets):
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache must be a PagedCache, got {type(cache).__name__}")
    _index("page_table", page_table, cache.device, 2)
    n = page_table.shape[0]
    if n < 1 or page_table.shape[1] < 1:
        raise ValueError(f"page_table must have a row for each sequence and at least one column, got shape "
                         f"{tuple(page_table.shape)}")
    _index(what, lengths, cache.device, 1)
    if lengths.shape[0] != n:
        raise ValueError(f"{what} must have one entry for each of {n} sequences, got {lengths.shape[0]}")
    if offsets is not None:
        _index("offsets", offsets, cache.device, 1)
        if offsets.shape[0] != n + 1:
            raise ValueError(f"offsets must have {n + 1} entries, got {offsets.shape[0]}")


def _scale(value) -> float:
    try:
        if isinstance(value, str):
            raise TypeError
        scale = float(value)
    except TypeError:
        raise TypeError(f"scale must be a number, got {type(value).__name__}") from None
    except OverflowError:
        scale = math.inf
    if not 0.0 <= scale <= torch.finfo(torch.float32).max:
        raise ValueError(f"scale must be finite in 32 bits and not negative, got {value}")
    return scale


def _no_gradient(name, t):
    if t.requires_grad and torch.is_grad_enabled() or has_tangent(t):
        raise ValueError(f"the cache does not take part in autograd, but {name} does: detach it, or run under "
                         "torch.no_grad()")


def _gpu(cache):
    if not device_ready():
        raise RuntimeError("no ROCm GPU available; cannot run the cache kernels")
    if cache.device.type != "cuda":
        raise ValueError(f"the cache must be on the GPU (device='cuda'), got {cache.device}")


def _on_device(device, fn, *args):
    dev = device.index if device.index is not None else torch.cuda.current_device()
    if current_device() == dev:
        return fn(*args, stream_handle(dev))
    with device_context(dev):
        return fn(*args, stream_handle(dev))


def append_paged_cache(cache: PagedCache, k, v, page_table, starts, *, offsets=None, rotary: RotaryPlan | None = None,
                       q=None):
    """Write new keys and values ``(tokens, kv_heads, head_dim)`` (float32,
    float16 or bfloat16, any strides with adjacent channels) to the cache.

    Sequence ``b``'s tokens are rows ``offsets[b] .. offsets[b + 1]`` (None:
    one token a sequence; rows before the first offset and past the last are
    padding) and take the positions from ``starts[b]`` on, in the pages
    ``page_table[b]`` names.  With ``rotary`` the keys are rotated by
    their positions first, and ``q`` ``(tokens, q_heads, head_dim)``, if
    given, is rotated in the same launch and returned (without ``rotary``:
    copied).

    A token in a page's first slot opens the page anew.  A page whose later
    tokens need a larger scale has its codes rescaled.  Infinities and
    NaN become NaN.  Tokens past the table's width, or whose page number is
    not one of the cache's, are skipped.  No page may belong to two sequences
    of one call.  ``page_table`` ``(sequences, width)``, ``starts`` and
    ``offsets`` are int32 on the cache's device.  Takes no part in autograd:
    tensors that require a gradient are refused unless under
    ``torch.no_grad()``.
    """
    _sequences(cache, page_table, starts, "starts", offsets)
    _heads("k", k, cache, heads=cache.kv_heads)
    _heads("v", v, cache, k.dtype, cache.kv_heads)
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError(f"k and v must have as many tokens, got {tokens} and {v.shape[0]}")
    if offsets is None and tokens != starts.shape[0]:
        raise ValueError(f"without offsets each sequence takes one token: got {tokens} tokens for "
                         f"{starts.shape[0]} sequences")
    out, qs, os, heads = None, (0, 0), (0, 0), 0
    if q is not None:
        _heads("q", q, cache, k.dtype)
        if q.shape[0] != tokens:
            raise ValueError(f"q must have as many tokens as k, got {q.shape[0]} and {tokens}")
        heads = q.shape[1]
    if rotary is not None:
        if not isinstance(rotary, RotaryPlan):
            raise TypeError(f"rotary must be a RotaryPlan, got {type(rotary).__name__}")
        if rotary.head_dim != cache.head_dim:
            raise ValueError(f"the rotary plan is for head_dim {rotary.head_dim}, the cache has {cache.head_dim}")
    _no_gradient("k", k)
    _no_gradient("v", v)
    if q is not None:
        _no_gradient("q", q)
    _gpu(cache)
    if q is not None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qs, os = q.stride(), out.stride()
    ks, vs = k.stride(), v.stride()
    args = native.APPEND_ARGS.pack(
        k.data_ptr(), v.data_ptr(), q.data_ptr() if heads else 0, out.data_ptr() if heads else 0, ks[0], ks[1], vs[0],
        vs[1], qs[0], qs[1], os[0], os[1], page_table.data_ptr(), starts.data_ptr(),
        0 if offsets is None else offsets.data_ptr(), page_table.stride(0), tokens, page_table.shape[1],
        starts.shape[0], heads, _DTYPES[k.dtype])
    with _ledger.phase("cache-append"):
        _on_device(cache.device, native.cache_append, cache._packed,
                   None if rotary is None else rotary.native(k.get_device()), args)
    return out


def attend_paged_cache(cache: PagedCache, q, page_table, lengths, *, offsets=None, scale: float | None = None,
                       causal: bool = True, window: int | None = None, max_length: int | None = None,
                       return_lse: bool = False):
    """Attention of ``q`` ``(tokens, q_heads, head_dim)`` (float16 or bfloat16;
    ``q_heads`` a multiple of the cache's) over the cache: ``softmax(scale q k)
    v``, a new tensor of ``q``'s shape and type.  Scores, maxima and sums are
    held in 32 bits; the softmax's weights are rounded to ``q``'s type for the
    product with ``v``.  ``q`` must be 16-byte aligned, and its strides keep it so.

    Sequence ``b``'s queries are rows ``offsets[b] .. offsets[b + 1]`` (None:
    as many for every sequence) and are the last of its ``lengths[b]``
    positions.  ``causal``: a query sees the keys up to its own position;
    ``window``: only that many of the last ones.  A query that sees no key, or
    is no sequence's (padding before the first offset or past the last), gives 0.
    ``scale`` defaults to ``head_dim ** -0.5``.  ``max_length``, if given,
    bounds ``lengths`` and lets short calls run in one launch; a longer
    sequence is still computed.  ``return_lse``: also the logarithm of the sum
    of exponentials, float32 ``(tokens, q_heads)``, -inf for such a query.
    A sequence longer than its table's pages, or with a page number that is not
    one of the cache's, gives NaN.  Takes no part in autograd: a ``q`` that
    requires a gradient is refused unless under ``torch.no_grad()``.
    """
    _sequences(cache, page_table, lengths, "lengths", offsets)
    _heads("q", q, cache)
    if q.dtype is torch.float32:
        raise TypeError("q must be float16 or bfloat16, got torch.float32")
    tokens, heads = q.shape[0], q.shape[1]
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"q must have a multiple of the cache's {cache.kv_heads} heads, got {heads}")
    if offsets is None and tokens % lengths.shape[0]:
        raise ValueError(f"without offsets every sequence has as many queries: got {tokens} tokens for "
                         f"{lengths.shape[0]} sequences")
    if window is not None and (isinstance(window, bool) or not isinstance(window, int) or not 1 <= window <= _MAX_POSITIONS):
        raise ValueError(f"window must be None or an int in [1, {_MAX_POSITIONS}], got {window!r}")
    if max_length is not None and (isinstance(max_length, bool) or not isinstance(max_length, int) or max_length < 0):
        raise ValueError(f"max_length must be None or an int of at least 0, got {max_length!r}")
    scale = cache.head_dim ** -0.5 if scale is None else _scale(scale)
    _no_gradient("q", q)
    _gpu(cache)
    out = torch.empty((tokens, heads, cache.head_dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    qs, os = q.stride(), out.stride()

    def pack(ws, nbytes):
        return native.ATTEND_ARGS.pack(
            q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), qs[0], qs[1], os[0], os[1],
            page_table.data_ptr(), lengths.data_ptr(), 0 if offsets is None else offsets.data_ptr(),
            page_table.stride(0), tokens, page_table.shape[1], lengths.shape[0], heads, _DTYPES[q.dtype],
            scale, bool(causal), window or 0, 0 if max_length is None else min(max_length, _MAX_POSITIONS), ws, nbytes)

    with _ledger.phase("cache-attend"):
        args = pack(0, 0)
        need = native.cache_attend_workspace(cache._packed, args)
        if need:
            # this call's, from torch's stream-ordered allocator on this stream
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            args = pack(ws.data_ptr(), need)
        _on_device(cache.device, native.cache_attend, cache._packed, args)
    return (out, lse) if return_lse else out
