"""What the cache's operators do not differentiate they refuse: a tensor that
requires a gradient, or carries a forward-mode tangent, would come back without
one and a backward pass through the rest would be wrong."""
import pytest
import torch
from torch.autograd import forward_ad

from kunlunxin_fft_amd import PagedCache, append_paged_cache, attend_paged_cache

I32 = dict(dtype=torch.int32)


def _append(**change):
    kw = dict(cache=PagedCache.empty(4, 2, 64, 16, device="cpu"), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64),
              q=torch.zeros(3, 4, 64), page_table=torch.zeros(3, 2, **I32), starts=torch.zeros(3, **I32))
    return append_paged_cache(**{**kw, **change})


def _attend(q):
    return attend_paged_cache(PagedCache.empty(4, 2, 64, 16, device="cpu"), q, torch.zeros(3, 2, **I32), torch.zeros(3, **I32))


def _calls():
    wanted = torch.zeros(3, 2, 64, requires_grad=True)
    yield lambda t: _append(k=t), wanted
    yield lambda t: _append(v=t), wanted
    yield lambda t: _append(q=t), torch.zeros(3, 4, 64, requires_grad=True)
    yield _attend, torch.zeros(3, 4, 64, dtype=torch.bfloat16, requires_grad=True)


@pytest.mark.parametrize("which", range(4), ids=["append k", "append v", "append q", "attend q"])
def test_refuses_what_requires_a_gradient(which):
    call, t = list(_calls())[which]
    with pytest.raises(ValueError, match="autograd"):
        call(t)
    with pytest.raises(ValueError, match="autograd"):  # a view of it, as a projection's output is
        call(t * 1.0)


@pytest.mark.parametrize("which", range(4), ids=["append k", "append v", "append q", "attend q"])
def test_refuses_tangents(which):
    call, t = list(_calls())[which]
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="autograd"):
            call(forward_ad.make_dual(t.detach(), torch.ones_like(t)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="passes the checks and asks for the cache to be on the GPU")
@pytest.mark.parametrize("which", range(4), ids=["append k", "append v", "append q", "attend q"])
def test_takes_them_without_gradients(which):
    """Under no_grad, and detached, as a serving loop has them: the next check."""
    call, t = list(_calls())[which]
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        call(t)
    with pytest.raises(RuntimeError, match="GPU"):
        call(t.detach())
