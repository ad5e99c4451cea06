"""Attention in a window whose first tokens stay visible: every form of the
kernel, sinks before, beside and inside the window, sequences shorter than
them, pages in between that are others', NaN there and where it counts."""
import numpy as np
import pytest
import torch

import lm_more_oracle as more
import lm_oracle as lm
from kunlunxin_fft_amd import attend_paged_cache
from test_gpu_paged_cache import _f64, _filled, _i32, _randn

pytestmark = pytest.mark.gpu


def _check(cache, q, table, lengths, counts, dtype, window, sinks, **kw):
    dev = q.device
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), dev)
    out, lse = attend_paged_cache(cache, q, table, _i32(lengths, dev), offsets=off, return_lse=True, window=window, sinks=sinks, **kw)
    want, want_lse, bound = more.attend(lm.Cache.of(cache), _f64(q), table.cpu().numpy(), lengths, counts, q.shape[-1] ** -0.5,
                                        kw.get("causal", True), window, sinks, dtype)
    got, g = _f64(out), _f64(lse)
    off_by = np.abs(got - want)
    assert (off_by <= bound).all(), f"worst {np.nanmax(off_by / bound)} of the bound, {np.isnan(got).sum()} NaN"
    empty = np.isneginf(want_lse)
    assert (np.isneginf(g) == empty).all() and (got[empty] == 0).all()
    assert (np.abs(g[~empty] - want_lse[~empty]) <= 2.0 ** -16 * (1 + np.abs(want_lse[~empty]))).all()
    return out


CASES = [
    # (dim, kv heads, group, page, lengths, counts, window, sinks, dtype, options)
    (128, 1, 1, 16, [1], [1], 1, 1, "bf16", {}),
    (128, 2, 4, 64, [0, 1, 5, 63, 64, 65, 127, 128, 129, 300, 1000, 2111], [1] * 12, 50, 4, "bf16", {}),
    (64, 3, 7, 16, [0, 900, 33, 256], [1] * 4, 100, 1, "fp16", {}),
    (96, 1, 16, 32, [777, 500], [1] * 2, 64, 64, "bf16", {}),
    (96, 2, 3, 16, [777, 90], [1] * 2, 1, 130, "fp16", {}),
    (256, 2, 3, 48, [900, 48, 49], [1] * 3, 33, 65, "fp16", {}),
    (128, 1, 32, 128, [700, 4], [1] * 2, 128, 7, "bf16", {}),
    (64, 2, 8, 64, [830, 70, 9], [5] * 3, 90, 16, "bf16", {}),
    (128, 2, 2, 16, [500, 40, 3, 0, 66], [33, 1, 5, 2, 66], 20, 10, "fp16", {}),
    (64, 1, 4, 32, [700, 450], [90, 450], 37, 5, "bf16", {}),
    (64, 1, 4, 32, [700, 450], [90, 450], 37, 300, "fp16", {}),
    (96, 2, 1, 16, [470, 64, 2], [3] * 3, 1, 2, "fp16", {}),
    (128, 1, 5, 64, [300, 20], [4] * 2, 1000, 9, "bf16", {}),
    (64, 1, 2, 16, [490, 30], [70, 40], 20, 3, "bf16", {"causal": False}),
    (256, 1, 4, 64, [700, 329], [70, 329], 60, 100, "bf16", {}),
    (128, 2, 4, 32, [1200, 813], [200, 600], 100, 4, "bf16", {}),
    (128, 2, 4, 32, [1200, 813], [200, 600], 100, 4, "fp16", {}),
    (64, 4, 1, 16, [2500], [1], 2400, 90, "fp16", {}),
    (128, 1, 8, 64, [6000, 10, 700], [1] * 3, 2500, 70, "bf16", {"max_length": 6000}),
    (96, 1, 12, 16, [600, 330], [4, 4], 90, 20, "bf16", {}),
    (64, 1, 6, 16, [600, 330], [9, 9], 90, 20, "fp16", {}),
    (128, 1, 6, 16, [600, 330], [9, 9], 90, 20, "bf16", {}),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend(gpu, case):
    dim, heads, group, page, lengths, counts, window, sinks, dtype, kw = case
    print("sinks", case, flush=True)
    cache, table = _filled(gpu, lengths, heads, dim, page, dtype, 40, size=2.0)
    q = _randn((sum(counts), heads * group, dim), dtype, gpu, 41, 2.0)
    a = _check(cache, q, table, lengths, counts, dtype, window, sinks, **kw)
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), gpu)
    b = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, window=window, sinks=sinks, **kw)
    assert torch.equal(a, b)


@pytest.mark.parametrize("group,counts", [(1, [1, 1]), (20, [1, 1]), (40, [1, 1]), (2, [50, 1]), (4, [200, 30])], ids=str)
def test_pages_between_do_not_count(gpu, group, counts):
    """Pages that hold neither a sink nor a key of any window may be others':
    other numbers, none at all, or full of NaN under NaN scales."""
    lengths, window, sinks, page = [900, 700], 80, 20, 16
    cache, table = _filled(gpu, lengths, 1, 128, page, "bf16", 50)
    q = _randn((sum(counts), group, 128), "bf16", gpu, 51)
    off = _i32(lm.offsets_of(counts), gpu)
    want = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, window=window, sinks=sinks)
    _check(cache, q, table, lengths, counts, "bf16", window, sinks)
    free = table.clone()
    for b, (n, c) in enumerate(zip(lengths, counts)):
        first = max(0, n - c - window + 1) // page
        free[b, -(-sinks // page):first] = torch.tensor([-1, cache.pages, 1 << 30, -7] * 100, dtype=torch.int32, device=gpu)[:max(0, first - -(-sinks // page))]
    assert not torch.equal(free, table)
    assert torch.equal(attend_paged_cache(cache, q, free, _i32(lengths, gpu), offsets=off, window=window, sinks=sinks), want)
    spoiled = int(table[0, 5])
    cache.k.view(torch.uint8)[spoiled] = 0x7f
    cache.v.view(torch.uint8)[spoiled] = 0xff
    cache.k_scale[spoiled] = cache.v_scale[spoiled] = float("nan")
    assert torch.equal(attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, window=window, sinks=sinks), want)


@pytest.mark.parametrize("group", [1, 40])
@pytest.mark.parametrize("n", [1, 60, 300])
def test_nan_counts_only_where_seen(gpu, n, group):
    """A NaN value in a sink reaches every query, in its channel; past the
    sinks and before the windows, none; a NaN key all channels."""
    length, window, sinks = 500, 40, 5
    cache, table = _filled(gpu, [length], 1, 64, 16, "bf16", 80)
    q = _randn((n, group, 64), "bf16", gpu, 81)
    off = _i32([0, n], gpu)
    want, _, bound = more.attend(lm.Cache.of(cache), _f64(q), table.cpu().numpy(), [length], [n], 64 ** -0.5, True, window, sinks)
    v, k = cache.v.view(torch.uint8), cache.k.view(torch.uint8)

    def run():
        return _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=off, window=window, sinks=sinks))

    for key, seen in ((3, True), (sinks, False), (100, False)):
        page, slot = int(table[0, key // 16]), key % 16
        # the windows that reach the key itself
        direct = np.array([length - n + i - window < key <= length - n + i for i in range(n)])
        after = np.array([key <= length - n + i for i in range(n)])
        rows = (after if seen else np.zeros(n, bool)) | direct
        keep = v[page, 0, 0, 9, slot].item()
        v[page, 0, 0, 9, slot] = 0x7f
        got = run()
        assert np.isnan(got[rows, :, 9]).all()
        got[rows, :, 9] = want[rows, :, 9]
        assert (np.abs(got - want) <= bound).all()
        v[page, 0, 0, 9, slot] = keep
        keep = k[page, 0, slot, 9].item()
        k[page, 0, slot, 9] = 0xff
        got = run()
        assert np.isnan(got[rows]).all()
        got[rows] = want[rows]
        assert (np.abs(got - want) <= bound).all()
        k[page, 0, slot, 9] = keep


def test_a_window_over_everything_is_none(gpu):
    lengths = [700, 64, 1]
    cache, table = _filled(gpu, lengths, 2, 128, 64, "bf16", 60)
    q = _randn((3, 8, 128), "bf16", gpu, 61)
    want, _, bound = lm.attend(lm.Cache.of(cache), _f64(q), table.cpu().numpy(), lengths, [1] * 3, 128 ** -0.5)
    for window, sinks in ((700, 4), (1, 700), (1 << 30, 1 << 30), (300, 400), (301, 399), (650, 600)):
        got = _f64(attend_paged_cache(cache, q, table, _i32(lengths, gpu), window=window, sinks=sinks))
        assert (np.abs(got - want) <= bound).all(), (window, sinks)
    a = attend_paged_cache(cache, q, table, _i32(lengths, gpu))
    assert torch.equal(attend_paged_cache(cache, q, table, _i32(lengths, gpu), sinks=9), a)
    a = attend_paged_cache(cache, q, table, _i32(lengths, gpu), window=90)
    assert torch.equal(attend_paged_cache(cache, q, table, _i32(lengths, gpu), window=90, sinks=0), a)


@pytest.mark.parametrize("size", [300.0, 3e4], ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_scores(gpu, dtype, size):
    """Scores far past where their differences are taken in one step: a sink
    that has the largest outweighs the window, whichever comes first."""
    length, dim = 2000, 64
    cache, table = _filled(gpu, [length], 1, dim, 16, dtype, 70)
    q = _randn((1, 2, dim), dtype, gpu, 71)
    k, _ = lm.Cache.of(cache).tokens(table[0].tolist(), length)
    keys = [0, 1, 2, length - 30, length - 1]
    s = np.einsum("hd,kd->hk", _f64(q)[0], k[keys, 0])
    for h in range(2):
        assert len(set(s[h])) == 5
    got = _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), window=30, sinks=3, scale=size))[0]
    kk, vv = lm.Cache.of(cache).tokens(table[0].tolist(), length)
    seen = [0, 1, 2] + list(range(length - 30, length))
    s = _f64(q)[0] @ kk[seen, 0].T * size
    order = np.sort(s, 1)
    # the runner-up is e^-20 or less of it, below half a step of either type
    assert (order[:, -1] - order[:, -2] > 20).all()
    want = vv[seen, 0][s.argmax(1)]
    u = lm.HALF_ULP[dtype]
    assert (np.abs(got - want) <= 2 * u * np.abs(want) + 2 * u).all()


def test_padding_bad_pages_and_graph(gpu):
    """Rows of no sequence give 0; a bad page that is seen NaN; a captured step
    whose lengths move, so that the sinks and the window part."""
    lengths = [400, 90]
    cache, table = _filled(gpu, [n + 300 for n in lengths], 2, 128, 16, "bf16", 90)
    q = _randn((7, 8, 128), "bf16", gpu, 91)
    out = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=_i32([2, 3, 5], gpu), window=50, sinks=4)
    assert bool((out[[0, 1, 5, 6]] == 0).all()) and torch.isfinite(out).all() and bool((out[2:5] != 0).any())
    bad = table.clone()
    bad[0, 0] = -1
    out = attend_paged_cache(cache, q[:2], bad, _i32(lengths, gpu), window=50, sinks=4)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    q, now = q[:2], _i32([40, 70], gpu)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        attend_paged_cache(cache, q, table, now, window=50, sinks=4)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = attend_paged_cache(cache, q, table, now, window=50, sinks=4)
    torch.cuda.synchronize()
    for _ in range(4):
        now += 71
        q.copy_(_randn((2, 8, 128), "bf16", gpu, int(now[0])))
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, _check(cache, q, table, now.tolist(), [1, 1], "bf16", 50, 4))
    del graph
