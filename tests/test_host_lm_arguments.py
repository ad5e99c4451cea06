"""What the language-model operators accept and refuse, before any device work."""
import copy

import pytest
import torch

from kunlunxin_fft_amd import PagedCache, attend_paged_cache, native


def _cache():
    return PagedCache.empty(4, 2, 64, 16, device="cpu")


def test_a_caches_tensors_stay():
    """The addresses the kernels use are taken once: another tensor, or none,
    cannot be put in a cache's place."""
    c = _cache()
    for name in ("k", "v", "k_scale", "v_scale", "pages", "device"):
        with pytest.raises(AttributeError, match="PagedCache"):
            setattr(c, name, getattr(c, name))
        with pytest.raises(AttributeError, match="PagedCache"):
            delattr(c, name)


def test_a_copy_of_a_cache_is_of_its_own_tensors():
    c = _cache()
    for d, shared in ((copy.copy(c), True), (copy.deepcopy(c), False)):
        assert native.CACHE_ARGS.unpack(d._packed)[:4] == (d.k.data_ptr(), d.v.data_ptr(), d.k_scale.data_ptr(), d.v_scale.data_ptr())
        assert (d.k.data_ptr() == c.k.data_ptr()) is shared
        assert (d.pages, d.kv_heads, d.page_size, d.head_dim) == (c.pages, c.kv_heads, c.page_size, c.head_dim)


def _attend(**kw):
    i32 = dict(dtype=torch.int32)
    return attend_paged_cache(_cache(), torch.zeros(3, 4, 64).half(), torch.zeros(3, 2, **i32), torch.zeros(3, **i32), **kw)


@pytest.mark.parametrize("kw,error", [
    ({"scale": "0.1"}, TypeError), ({"scale": [0.1]}, TypeError), ({"scale": 1j}, TypeError),
    ({"scale": float("nan")}, ValueError), ({"scale": float("inf")}, ValueError), ({"scale": -0.5}, ValueError),
    ({"scale": 1e39}, ValueError), ({"scale": 10 ** 400}, ValueError), ({"window": (1 << 30) + 1}, ValueError),
    ({"window": 1 << 70}, ValueError), ({"max_length": 1.0}, ValueError),
], ids=lambda v: str(v)[:24])
def test_attend_refuses(kw, error):
    """In the framework's errors, and before a GPU is asked for."""
    with pytest.raises(error, match=next(iter(kw))):
        _attend(**kw)


@pytest.mark.skipif(torch.cuda.is_available(), reason="passes the checks and asks for the cache to be on the GPU")
@pytest.mark.parametrize("kw", [{"scale": 1}, {"scale": 0.0}, {"scale": torch.tensor(0.5)}, {"window": 1 << 30},
                                {"max_length": 1 << 70}], ids=str)
def test_attend_takes(kw):
    with pytest.raises(RuntimeError, match="GPU"):
        _attend(**kw)


def test_a_length_bound_past_64_bits_is_none(monkeypatch):
    """max_length only bounds: one that no sequence can reach packs as the
    largest table does."""
    from kunlunxin_fft_amd import paged_cache

    packed = []
    monkeypatch.setattr(paged_cache, "_gpu", lambda cache: None)
    monkeypatch.setattr(native, "cache_attend_workspace", lambda cache, args: packed.append(native.ATTEND_ARGS.unpack(args)) or 0)
    monkeypatch.setattr(paged_cache, "_on_device", lambda *a: None)
    _attend(max_length=1 << 70)
    assert packed[0][19] == 1 << 30
    _attend(max_length=77)
    assert packed[1][19] == 77
