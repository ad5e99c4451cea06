"""Attention in a window with sinks where items are cut over several workgroups:
every form of the kernel in both types, parts that begin inside the sinks,
inside the windows and between, pages between them that are others', NaN."""
import pytest
import torch

import lm_device_oracle as dev
import lm_oracle as lm
from kunlunxin_fft_amd import attend_paged_cache, native
from test_gpu_paged_cache import _filled, _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture
def workspaces(monkeypatch):
    """The bytes of workspace that each call asked for: a call whose items are
    whole needs none."""
    real, seen = native.cache_attend_with_workspace, []
    monkeypatch.setattr(native, "cache_attend_with_workspace", lambda *a: seen.append(real(*a)) or seen[-1])
    return seen


CASES = [
    # (dim, kv heads, group, page, lengths, counts, window, sinks, causal): by rows a sequence and key head
    (256, 1, 5, 64, [2900, 2500], [1, 1], 2400, 70, True),           # to 16
    (96, 2, 7, 32, [2700, 900, 3000], [1, 2, 2], 2400, 300, True),
    (64, 1, 20, 16, [3100], [1], 2500, 300, True),                   # to 32
    (128, 2, 8, 32, [3100, 2700, 5], [3, 3, 3], 2450, 70, True),
    (64, 1, 8, 64, [2800, 3100], [6, 6], 2400, 130, True),           # to 64
    (96, 1, 12, 16, [3100], [4], 2500, 70, True),
    (128, 1, 8, 48, [3100, 2600], [7, 4], 2400, 130, True),
    (128, 2, 8, 64, [40000, 5000], [7, 7], 2500, 1000, True),
    (256, 1, 4, 64, [2800], [40], 2400, 70, True),                   # head dim 256, many
    (256, 2, 3, 16, [3100, 2600, 0], [50, 7, 30], 900, 1700, True),
    (64, 1, 4, 32, [3100], [90], 2300, 200, True),                   # more
    (96, 1, 3, 16, [3100, 100], [70, 60], 500, 2100, True),
    (128, 1, 4, 64, [5000, 2700], [60, 150], 2500, 70, True),
    (128, 2, 4, 32, [9000], [300], 2400, 65, True),
    (64, 1, 2, 16, [2600, 1500], [50, 40], 700, 130, False),
    (128, 1, 4, 16, [2000], [1], 300, 70, False),
    (256, 1, 4, 64, [1900, 2300], [9, 20], 300, 200, False),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend(gpu, case, dtype, workspaces):
    dim, heads, group, page, lengths, counts, window, sinks, causal = case
    print("sinks, cut", case, dtype, flush=True)
    cache, table = _filled(gpu, lengths, heads, dim, page, dtype, 140, size=2.0)
    off = _i32(lm.offsets_of(counts), gpu)
    for size in (2.0, 30.0):  # the latter: a few keys have all the weight
        q = _randn((sum(counts), heads * group, dim), dtype, gpu, 141, size)
        kw = dict(offsets=off, window=window, sinks=sinks, causal=causal)
        out, lse = attend_paged_cache(cache, q, table, _i32(lengths, gpu), return_lse=True, **kw)
        assert workspaces[-1] > 0
        dev.check_attend(out, lse, dev.attend(cache, q, table, lengths, counts, causal=causal, window=window, sinks=sinks))
        assert torch.equal(attend_paged_cache(cache, q, table, _i32(lengths, gpu), **kw), out)  # the same bits every time


FORMS = [(64, 4, 1), (128, 20, 1), (64, 10, 5), (128, 10, 5), (256, 4, 60), (64, 4, 60), (128, 2, 200)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group,n", FORMS, ids=str)
def test_pages_between_do_not_count(gpu, dim, group, n, dtype, workspaces):
    length, window, sinks, page = 6000, 2500, 150, 16
    cache, table = _filled(gpu, [length], 1, dim, page, dtype, 150)
    q = _randn((n, group, dim), dtype, gpu, 151)
    kw = dict(offsets=_i32([0, n], gpu), window=window, sinks=sinks)
    want, lse = attend_paged_cache(cache, q, table, _i32([length], gpu), return_lse=True, **kw)
    assert workspaces[-1] > 0
    dev.check_attend(want, lse, dev.attend(cache, q, table, [length], [n], window=window, sinks=sinks))
    first, last = -(-sinks // page), (length - n - window + 1) // page
    spoiled = table[0, first:last].long()
    for t in (cache.k, cache.v):
        t.view(torch.uint8)[spoiled] = 0x7f
    cache.k_scale[spoiled] = cache.v_scale[spoiled] = float("nan")
    assert torch.equal(attend_paged_cache(cache, q, table, _i32([length], gpu), **kw), want)
    free = table.clone()
    free[0, first:last] = torch.tensor([-1, cache.pages, 1 << 30, -7] * 100, dtype=torch.int32, device=gpu)[:last - first]
    assert torch.equal(attend_paged_cache(cache, q, free, _i32([length], gpu), **kw), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group,n", FORMS, ids=str)
def test_nan_counts_only_where_seen(gpu, dim, group, n, dtype, workspaces):
    """A NaN value in a sink, past the sinks, at both ends of the windows and in
    their middle reaches the queries that see it, in its channel; a NaN key all
    their channels."""
    length, window, sinks = 2900, 2450, 150
    cache, table = _filled(gpu, [length], 1, dim, 16, dtype, 160)
    q = _randn((n, group, dim), dtype, gpu, 161)
    want, _, bound = dev.attend(cache, q, table, [length], [n], window=window, sinks=sinks)
    v, k = cache.v.view(torch.uint8), cache.k.view(torch.uint8)
    pos = torch.arange(length - n, length, device=gpu)
    # between the sinks and every window; the first and last that some window has
    for key in (3, sinks - 1, sinks, length - n - window, length - n - window + 1, length - window, 1500, length - n, length - 1):
        seen = (key <= pos) & ((key > pos - window) | (key < sinks))
        page, slot = int(table[0, key // 16]), key % 16
        for codes, at, channel in ((v, (page, 0, 0, 9, slot), 9), (k, (page, 0, slot, 9), slice(None))):
            keep = codes[at].item()
            codes[at] = 0x7f
            got = attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu), window=window, sinks=sinks).double()
            assert workspaces[-1] > 0
            assert bool(got[seen][..., channel].isnan().all()), key
            hit = torch.zeros_like(got, dtype=torch.bool)
            hit[seen.nonzero()[:, 0][:, None], :, torch.arange(dim, device=gpu)[channel].reshape(1, -1)] = True
            assert bool(((got - want).abs() <= bound)[~hit].all()), key
            codes[at] = keep
