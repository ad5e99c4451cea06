"""The paged cache at its largest pages (more keys than a workgroup holds at once,
64 units of sixteen a page) and over more sequences than a wave looks at together."""
import numpy as np
import pytest

import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, plan_rotary
from test_gpu_paged_cache import _check, _f64, _filled, _i32, _randn, _same, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rot,layout", [(None, None), ("all", "half"), (32, "interleaved")])
@pytest.mark.parametrize("dim,page,dtype", [(256, 128, "bf16"), (128, 128, "fp32"), (64, 1024, "fp16"), (256, 1024, "fp32")])
def test_append_of_large_pages(gpu, dim, page, dtype, rot, layout):
    """Whole pages, and pieces that start inside one and end off a unit of sixteen."""
    print("append", dim, page, dtype, rot, layout, flush=True)
    heads, starts, counts = 2, [0, 37, page - 5, 3 * page], [2 * page, page + 3, 11, 0]
    plan = None if rot is None else plan_rotary(dim, rot_dim=dim if rot == "all" else rot, layout=layout)
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 400)
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    want, rows = lm.Cache.of(cache), table.cpu().numpy()
    for first, new, size, seed in ((0 * np.array(starts), starts, 1.0, 401), (starts, counts, 3.0, 403)):
        t = int(sum(new))
        k, v = (_randn((t, heads, dim), dtype, gpu, s, size) for s in (seed, seed + 1))
        append_paged_cache(cache, k, v, table, _i32(list(map(int, first)), gpu),
                           offsets=_i32(lm.offsets_of(new), gpu), rotary=plan)
        kr = _f64(k)
        if plan is not None:
            pos = np.concatenate([np.arange(a, a + n) for a, n in zip(first, new)])
            kr = lm.rotate(kr, pos, plan.frequencies, layout)
        want.append(kr, _f64(v), rows, [int(a) for a in first], new)
        # rotated pages that grow round codes again: what a neighbouring code became
        got = lm.Cache.of(cache)
        assert np.isfinite(got.k).all() and np.isfinite(got.v).all()
        _same(cache, want, exact_k=plan is None)


@pytest.mark.parametrize("dim,group,n", [(64, 1, 1), (128, 4, 6), (64, 4, 12), (256, 4, 12), (128, 4, 30)])
@pytest.mark.parametrize("length", [1500, 3000])
def test_attend_over_large_pages(gpu, dim, group, n, length):
    print("attend", dim, group, n, length, flush=True)
    cache, table = _filled(gpu, [length, n + 5], 1, dim, 1024, "bf16", 410)
    q = _randn((2 * n, group, dim), "bf16", gpu, 411)
    _check(cache, q, table, [length, n + 5], [n, n], "bf16")
    _check(cache, q, table, [length, n + 5], [n, n], "bf16", window=700)


def _many(count, longest, seed):
    r = np.random.default_rng(seed)
    lengths = r.integers(0, 40, count)
    lengths[r.integers(0, count, count // 8)] = 0
    lengths[[0, 63, 64, count - 1]] = [longest, 33, longest // 2, longest]
    return [int(n) for n in lengths]


@pytest.mark.parametrize("count", [65, 130, 256])
@pytest.mark.parametrize("max_length", [None, 60])
@pytest.mark.parametrize("new", [1, 3, "mixed", "queries in one"])
def test_many_sequences(gpu, count, max_length, new):
    """More than 64, empty ones among them, in one launch (max_length) and cut."""
    print("many", count, max_length, new, flush=True)
    longest = 60 if max_length else 2000
    lengths = _many(count, longest, 420)
    if isinstance(new, int):
        counts = [new] * count
    elif new == "mixed":
        counts = [int(min(n, c)) for n, c in zip(lengths, np.random.default_rng(421).integers(0, 9, count))]
    else:  # a prompt behind sequences without queries
        counts = [0] * count
        counts[-1] = 50
    cache, table = _filled(gpu, lengths, 2, 64, 16, "bf16", 422, width=130)
    q = _randn((sum(counts), 4, 64), "bf16", gpu, 423)
    _check(cache, q, table, lengths, counts, "bf16", **({"max_length": max_length} if max_length else {}))


@pytest.mark.parametrize("count", [70, 200])
def test_append_to_many_sequences(gpu, count):
    r = np.random.default_rng(430)
    starts, counts = [int(n) for n in r.integers(0, 50, count)], [int(n) for n in r.integers(0, 40, count)]
    table, pool = _table([a + n for a, n in zip(starts, counts)], 16, gpu, 431)
    cache = PagedCache.empty(pool, 2, 64, 16, gpu)
    want, rows = lm.Cache.of(cache), table.cpu().numpy()
    for first, new, seed in (([0] * count, starts, 432), (starts, counts, 434)):
        k, v = (_randn((sum(new), 2, 64), "fp16", gpu, s) for s in (seed, seed + 1))
        append_paged_cache(cache, k, v, table, _i32(first, gpu), offsets=_i32(lm.offsets_of(new), gpu))
        want.append(_f64(k), _f64(v), rows, first, new)
        _same(cache, want)


@pytest.mark.parametrize("dim,dtype", [(128, "bf16"), (64, "fp32")])
def test_append_of_a_padded_batch(gpu, dim, dtype):
    """Rows before the first offset and past the last are not cached."""
    counts, starts, before, after = [20, 0, 33], [5, 9, 0], 4, 70
    table, pool = _table([a + n for a, n in zip(starts, counts)], 16, gpu, 440)
    cache, own = (PagedCache.empty(pool, 2, dim, 16, gpu) for _ in range(2))
    off = _i32(lm.offsets_of(counts), gpu)
    k, v = (_randn((before + 53 + after, 2, dim), dtype, gpu, s) for s in (441, 442))
    append_paged_cache(cache, k, v, table, _i32(starts, gpu), offsets=off + before)
    append_paged_cache(own, k[before:before + 53], v[before:before + 53], table, _i32(starts, gpu), offsets=off)
    _same(cache, lm.Cache.of(own))
