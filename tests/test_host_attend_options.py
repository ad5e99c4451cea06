"""Sinks and shared prefixes without a GPU: the argument struct, and what
attention refuses before any device work."""
import pytest
import torch

from kunlunxin_fft_amd import PagedCache, attend_paged_cache, native
from test_host_lm_axes import check_layout

I32 = dict(dtype=torch.int32)


def _attend(**kw):
    return attend_paged_cache(PagedCache.empty(4, 2, 64, 16, device="cpu"), torch.zeros(3, 4, 64).half(), torch.zeros(3, 2, **I32),
                              torch.zeros(3, **I32), **kw)


@pytest.mark.parametrize("kw,error,text", [
    (dict(sinks=-1), ValueError, "sinks"), (dict(sinks=True), ValueError, "sinks"), (dict(sinks=4.0), ValueError, "sinks"),
    (dict(sinks=None), ValueError, "sinks"), (dict(sinks=(1 << 30) + 1, window=4), ValueError, "sinks"),
    (dict(prefix_pages=[1]), TypeError, "prefix_pages"), (dict(prefix_pages=torch.ones(1)), TypeError, "prefix_pages"),
    (dict(prefix_pages=torch.ones(1, dtype=torch.int64)), TypeError, "prefix_pages"),
    (dict(prefix_pages=torch.ones((), **I32)), ValueError, "prefix_pages"), (dict(prefix_pages=torch.ones(0, **I32)), ValueError, "prefix_pages"),
    (dict(prefix_pages=torch.ones(2, **I32)), ValueError, "prefix_pages"),
    (dict(prefix_pages=torch.ones(1, device="meta", **I32)), ValueError, "like the cache"),
    (dict(prefix_groups=torch.zeros(2, **I32)), ValueError, "give prefix_pages"),
    (dict(prefix_pages=torch.ones(2, **I32), prefix_groups=torch.zeros(2, **I32)), ValueError, "3 entries"),
    (dict(prefix_pages=torch.ones(1, **I32), prefix_groups=torch.zeros(2)), TypeError, "prefix_groups"),
    (dict(prefix_pages=torch.ones(4, **I32)[::2], prefix_groups=torch.zeros(3, **I32)), ValueError, "adjacent"),
], ids=str)
def test_refuses(kw, error, text):
    with pytest.raises(error, match=text):
        _attend(**kw)


@pytest.mark.skipif(torch.cuda.is_available(), reason="passes the checks and asks for the cache to be on the GPU")
@pytest.mark.parametrize("kw", [
    dict(sinks=0), dict(sinks=4), dict(sinks=1 << 30, window=1), dict(prefix_pages=torch.ones(1, **I32)),
    dict(prefix_pages=torch.ones(2, **I32), prefix_groups=torch.zeros(3, **I32)),
    dict(prefix_pages=torch.ones(1, **I32), window=3, sinks=2)], ids=str)
def test_takes(kw):
    with pytest.raises(RuntimeError, match="GPU"):
        _attend(**kw)


def test_options_struct_matches_the_header(tmp_path):
    check_layout(tmp_path, "mfft_attend_options", native.ATTEND_OPTIONS)


def test_calls_without_options_are_the_calls_they_were(monkeypatch):
    """And with them the options hold what was given."""
    from kunlunxin_fft_amd import paged_cache

    seen = []
    monkeypatch.setattr(paged_cache, "_gpu", lambda cache: None)
    monkeypatch.setattr(paged_cache, "_on_device", lambda device, fn, *a: seen.append((fn.__name__, a[2:])))
    monkeypatch.setattr(native, "cache_attend_workspace", lambda cache, args: 0)
    monkeypatch.setattr(native, "cache_attend_with_workspace", lambda cache, args, options: 0)
    pages, groups = torch.ones(2, **I32), torch.zeros(3, **I32)
    _attend(window=5)
    _attend(window=5, sinks=3)
    _attend(prefix_pages=pages, prefix_groups=groups)
    assert [s[0] for s in seen] == ["cache_attend", "cache_attend_with", "cache_attend_with"]
    assert native.ATTEND_OPTIONS.unpack(seen[1][1][0]) == (3, 0, 0, 0)
    assert native.ATTEND_OPTIONS.unpack(seen[2][1][0]) == (0, pages.data_ptr(), groups.data_ptr(), 2)


def test_c_entries_refuse_before_device_work():
    """The C entries' own checks (made-up addresses, never touched)."""
    lib = native.load()
    p = 1 << 20
    cache = native.CACHE_ARGS.pack(p, p, p, p, 4, 2, 64, 16)
    args = native.ATTEND_ARGS.pack(p, p << 10, 0, 128, 64, 128, 64, p, p, 0, 2, 3, 2, 3, 2, native.F16, 0.125, 1, 0, 0, 0, 0)
    for options, text in ((None, b"options"), ((-1, 0, 0, 0), b"sinks"), (((1 << 30) + 1, 0, 0, 0), b"sinks"), ((0, p, 0, 0), b"group"),
                          ((0, p, 0, 2), b"group"), ((0, p + 1, 0, 1), b"aligned"), ((0, p, p + 2, 2), b"aligned"), ((0, 0, p, 1), b"prefix_pages")):
        packed = None if options is None else native.ATTEND_OPTIONS.pack(*options)
        assert lib.mfft_cache_attend_with(cache, args, packed, None) == native.ERR_VALUE, options
        assert text in lib.mfft_last_error(), (options, lib.mfft_last_error())
        with pytest.raises(ValueError):
            native.cache_attend_with_workspace(cache, args, packed)
    # what is needed follows from the shapes: a row of the prefix for each query row
    need = native.cache_attend_with_workspace(cache, args, native.ATTEND_OPTIONS.pack(0, p, 0, 1))
    assert need >= 3 * 2 * (4 * 64 + 8)
    with pytest.raises(ValueError, match="workspace"):
        native.cache_attend_with(cache, args, native.ATTEND_OPTIONS.pack(0, p, 0, 1), 0)
    # a window and a prefix: the prefix is not used
    windowed = native.ATTEND_ARGS.pack(p, p << 10, 0, 128, 64, 128, 64, p, p, 0, 2, 3, 2, 3, 2, native.F16, 0.125, 1, 9, 0, 0, 0)
    assert native.cache_attend_with_workspace(cache, windowed, native.ATTEND_OPTIONS.pack(0, p, 0, 1)) == native.cache_attend_workspace(cache, windowed)
