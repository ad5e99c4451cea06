"""What the language-model operators accept and refuse, before any device work."""
import copy

import pytest

from kunlunxin_fft_amd import PagedCache, native


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
