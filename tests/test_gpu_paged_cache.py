"""The paged 8-bit cache: appending against the 64-bit form, and attention
over it: types, head layouts, lengths from none to long, pages that end inside
a tile, masks that leave a row nothing, NaN in masked places, bad indexes."""
import numpy as np
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, attend_paged_cache, plan_rotary

pytestmark = pytest.mark.gpu


def _f64(t):
    return t.detach().double().cpu().numpy()


def _randn(shape, dtype, gpu, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * size).to(lm.DTYPES[dtype]).to(gpu)


def _table(lengths, page, gpu, seed, spare=2, width=None):
    """Pages in random order, unused entries -1; (table, pages in the pool)."""
    need = [-(-int(n) // page) for n in lengths]
    pool = sum(need) + spare
    order = np.random.default_rng(seed).permutation(pool)
    t = np.full((len(need), width or max(1, max(need))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(t).to(gpu), pool


def _i32(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _same(cache, want, exact_k=True):
    """The cache's codes and scales against the oracle's; with rotated keys a
    32-bit rotation may round a code the other way, so those are compared as
    values, within the rounding's half step."""
    got = lm.Cache.of(cache)
    np.testing.assert_array_equal(got.vs, want.vs)
    np.testing.assert_array_equal(got.ks, want.ks)
    np.testing.assert_array_equal(got.v, want.v)
    if exact_k:
        np.testing.assert_array_equal(got.k, want.k)
    else:
        differ = got.k != want.k
        assert differ.mean() < 1e-3
        # a neighbouring code: one step, 2^-3 of its size or 2^-9
        assert (np.abs(got.k - want.k) <= np.maximum(np.abs(want.k) * 2.0 ** -3, 2.0 ** -9) * 1.01).all()


APPEND = [
    # (dim, kv heads, page, starts, counts, dtype)
    (128, 2, 64, [0], [1], "bf16"),
    (64, 1, 16, [5, 0, 16, 31], [1, 1, 1, 1], "fp16"),
    (96, 3, 32, [0, 7, 33], [100, 25, 1], "bf16"),
    (256, 1, 16, [15, 3], [2, 13], "fp32"),
    (128, 4, 128, [0, 127, 200], [300, 2, 56], "fp16"),
    (64, 8, 48, [10, 0, 47, 0], [0, 97, 50, 3], "fp32"),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, case):
    dim, heads, page, starts, counts, dtype = case
    print("append", case, flush=True)
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 1)
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    t, want = sum(counts), lm.Cache.of(cache)
    rows = table.cpu().numpy()
    if max(starts):  # what is cached before
        k, v = (_randn((sum(starts), heads, dim), dtype, gpu, s) for s in (2, 3))
        append_paged_cache(cache, k, v, table, _i32([0] * len(starts), gpu), offsets=_i32(lm.offsets_of(starts), gpu))
        want.append(_f64(k), _f64(v), rows, [0] * len(starts), starts)
        _same(cache, want)
    # larger values than before, so that half-filled pages grow
    k, v = (_randn((t, heads, dim), dtype, gpu, s, 5.0) for s in (4, 5))
    off = None if all(n == 1 for n in counts) else _i32(lm.offsets_of(counts), gpu)
    assert append_paged_cache(cache, k, v, table, _i32(starts, gpu), offsets=off) is None
    want.append(_f64(k), _f64(v), rows, starts, counts)
    _same(cache, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout,rot", [("half", 128), ("interleaved", 64), ("half", 20)])
def test_append_rotates(gpu, layout, rot, dtype):
    dim, heads, hq, page, starts, counts = 128, 2, 6, 32, [0, 40, 5], [70, 1, 0]
    plan = plan_rotary(dim, rot_dim=rot, layout=layout)
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 6)
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    want = lm.Cache.of(cache)
    t = sum(counts)
    fused = _randn((t, hq + 2 * heads, dim), dtype, gpu, 7)
    q, k, v = fused.split([hq, heads, heads], 1)
    got = append_paged_cache(cache, k, v, table, _i32(starts, gpu), offsets=_i32(lm.offsets_of(counts), gpu),
                             rotary=plan, q=q)
    pos = np.concatenate([np.arange(a, a + n) for a, n in zip(starts, counts)])
    kr = lm.rotate(_f64(k), pos, plan.frequencies, layout)
    want.append(kr, _f64(v), table.cpu().numpy(), starts, counts)
    _same(cache, want, exact_k=False)
    qr = lm.rotate(_f64(q), pos, plan.frequencies, layout)
    assert (np.abs(_f64(got) - qr) <= lm.rotate_bound(_f64(q), qr, dtype, plan.frequencies, layout)).all()


def test_append_token_by_token_keeps_codes(gpu):
    """A page filled one token at a time, each larger than the one before: the
    scale grows many times, and every value is still within one rounding (half
    a step of three fraction bits, 2^-4) of what was written, or a step of the
    least codes at each growth."""
    dim, page, n = 64, 16, 16
    cache = PagedCache.empty(1, 1, dim, page, gpu)
    table = _i32([[0]], gpu)
    want = lm.Cache.of(cache)
    xs = [_randn((1, 1, dim), "fp32", gpu, 30 + i, 1.7 ** i) for i in range(n)]
    for i, x in enumerate(xs):
        append_paged_cache(cache, x, x, table, _i32([i], gpu))
        want.append(_f64(x), _f64(x), [[0]], [i], [1])
    _same(cache, want)
    got = lm.Cache.of(cache)
    x = np.stack([_f64(x)[0, 0] for x in xs])
    err = np.abs(got.k[0, 0] * got.ks[0, 0] - x)
    assert (err <= 2.0 ** -4 * np.abs(x) + n * 2.0 ** -10 * got.ks[0, 0]).all()


def test_append_opens_pages_anew(gpu):
    """A recycled page: what it held, NaN codes and a huge scale, is gone."""
    cache = PagedCache.empty(1, 1, 64, 16, gpu)
    cache.k.view(torch.uint8).fill_(0x7f)
    cache.v.view(torch.uint8).fill_(0x7f)
    cache.k_scale.fill_(2.0 ** 100)
    cache.v_scale.fill_(2.0 ** 100)
    x = _randn((1, 1, 64), "bf16", gpu, 8)
    append_paged_cache(cache, x, x, _i32([[0]], gpu), _i32([0], gpu))
    s = lm.block_scale(_f64(x))
    assert cache.k_scale.item() == s and cache.v_scale.item() == s
    q = _randn((1, 1, 64), "bf16", gpu, 9)
    out = attend_paged_cache(cache, q, _i32([[0]], gpu), _i32([1], gpu))
    np.testing.assert_array_equal(_f64(out)[0, 0], lm.round_code(_f64(x)[0, 0] / s) * s)


def test_append_values_that_are_not_finite(gpu):
    cache = PagedCache.empty(1, 1, 64, 16, gpu)
    x = _randn((2, 1, 64), "fp32", gpu, 10)
    x[0, 0, 3], x[0, 0, 4], x[1, 0, 5] = float("inf"), -float("inf"), float("nan")
    y = x.clone()
    y[1] = float("nan")
    append_paged_cache(cache, x, y, _i32([[0]], gpu), _i32([0], gpu), offsets=_i32([0, 2], gpu))
    want = lm.Cache(*(np.zeros((1, 1, 16, 64)) for _ in range(2)), *(np.full((1, 1), 2.0 ** -126) for _ in range(2)))
    want.append(_f64(x), _f64(y), [[0]], [0], [2])
    _same(cache, want)


@pytest.mark.parametrize("size", [0.0, 2.0 ** -140, 3e38, 448.0, 448.0 * (1 + 2.0 ** -23)])
def test_append_extreme_sizes(gpu, size):
    cache = PagedCache.empty(1, 1, 64, 16, gpu)
    x = torch.full((1, 1, 64), size, device=gpu)
    x[0, 0, ::2] *= 0.5
    append_paged_cache(cache, x, -x, _i32([[0]], gpu), _i32([0], gpu))
    want = lm.Cache(*(np.zeros((1, 1, 16, 64)) for _ in range(2)), *(np.full((1, 1), 2.0 ** -126) for _ in range(2)))
    want.append(_f64(x), -_f64(x), [[0]], [0], [1])
    _same(cache, want)


def test_append_skips_what_has_no_page(gpu):
    """Page numbers out of range, and tokens past the table's width."""
    cache = PagedCache.empty(3, 2, 64, 16, gpu)
    before = lm.Cache.of(cache)
    k = _randn((3 * 20, 2, 64), "bf16", gpu, 11)
    table = _i32([[-1, 1], [3, 2], [1 << 30, 0]], gpu)
    append_paged_cache(cache, k, k, table, _i32([0, 0, 16], gpu), offsets=_i32([0, 20, 40, 60], gpu))
    before.append(_f64(k), _f64(k), table.cpu().numpy(), [0, 0, 16], [20, 20, 20])
    _same(cache, before)


def _filled(gpu, lengths, heads, dim, page, dtype, seed, width=None, size=1.0):
    table, pool = _table(lengths, page, gpu, seed, width=width)
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    # what no sequence holds is NaN
    cache.k.view(torch.uint8).fill_(0x7f)
    cache.v.view(torch.uint8).fill_(0xff)
    cache.k_scale.fill_(float("nan"))
    cache.v_scale.fill_(float("nan"))
    t = int(sum(lengths))
    k, v = (_randn((t, heads, dim), dtype, gpu, seed + i, size) for i in (1, 2))
    append_paged_cache(cache, k, v, table, _i32([0] * len(lengths), gpu),
                       offsets=_i32(lm.offsets_of([int(n) for n in lengths]), gpu))
    return cache, table


def _check(cache, q, table, lengths, counts, dtype, **kw):
    dev = q.device
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), dev)
    out, lse = attend_paged_cache(cache, q, table, _i32(lengths, dev), offsets=off, return_lse=True, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape
    scale = kw.get("scale") or q.shape[-1] ** -0.5
    want, want_lse, bound = lm.attend(lm.Cache.of(cache), _f64(q), table.cpu().numpy(), lengths, counts, scale,
                                      kw.get("causal", True), kw.get("window"), dtype)
    got = _f64(out)
    off_by = np.abs(got - want)
    assert (off_by <= bound).all(), f"worst {np.max(off_by / bound)} of the bound"
    empty = np.isneginf(want_lse)
    g = _f64(lse)
    assert (np.isneginf(g) == empty).all() and (got[empty] == 0).all()
    # the score's error, and 32-bit sums and logarithm
    assert (np.abs(g[~empty] - want_lse[~empty]) <= 2.0 ** -16 * (1 + np.abs(want_lse[~empty]))).all()
    return out


ATTEND = [
    # (dim, kv heads, group, page, lengths, counts, dtype, options)
    (128, 1, 1, 16, [1], [1], "bf16", {}),
    (128, 2, 4, 64, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000], [1] * 12, "bf16", {}),
    (64, 3, 7, 16, [0, 300, 33, 256], [1] * 4, "fp16", {}),
    (96, 1, 16, 32, [77, 500], [1] * 2, "bf16", {}),
    (256, 2, 3, 48, [200, 48, 49], [1] * 3, "fp16", {}),
    (128, 1, 32, 128, [400, 4], [1] * 2, "bf16", {}),
    (64, 2, 8, 64, [130, 70, 9], [5] * 3, "bf16", {}),
    (128, 2, 2, 16, [100, 40, 3, 0, 66], [33, 1, 5, 2, 66], "fp16", {}),
    (64, 1, 4, 32, [200, 150], [90, 150], "bf16", {"window": 37}),
    (96, 2, 1, 16, [170, 64, 2], [3] * 3, "fp16", {"window": 1}),
    (128, 1, 5, 64, [300, 20], [4] * 2, "bf16", {"window": 1000}),
    (64, 1, 2, 16, [90, 30], [70, 40], "bf16", {"causal": False}),
    (128, 1, 2, 64, [260, 0], [9] * 2, "fp16", {"causal": False, "window": 50}),
    (256, 1, 4, 64, [300, 129], [70, 129], "bf16", {}),
    (128, 2, 4, 32, [700, 513], [200, 300], "bf16", {"scale": 0.3}),
    (64, 4, 1, 16, [2500], [1], "fp16", {}),
    (128, 1, 8, 64, [3000, 10, 700], [1] * 3, "bf16", {"max_length": 3000}),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attend(gpu, case):
    dim, heads, group, page, lengths, counts, dtype, kw = case
    print("attend", case, flush=True)
    cache, table = _filled(gpu, lengths, heads, dim, page, dtype, 40, size=2.0)
    q = _randn((sum(counts), heads * group, dim), dtype, gpu, 41, 2.0)
    a = _check(cache, q, table, lengths, counts, dtype, **kw)
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), gpu)
    b = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, **kw)
    assert torch.equal(a, b)  # the same bits every time


def test_attend_more_queries_than_keys(gpu):
    """The first queries come before the first key: rows that see nothing."""
    cache, table = _filled(gpu, [5, 40], 1, 64, 16, "bf16", 50)
    q = _randn((12 + 60, 2, 64), "bf16", gpu, 51)
    _check(cache, q, table, [5, 40], [12, 60], "bf16")


def test_attend_long_context(gpu):
    """Long enough to be split over the chip, with a maximum that moves late."""
    n = 40000
    cache, table = _filled(gpu, [n, 17, 9000], 1, 64, 64, "bf16", 60)
    q = _randn((3, 2, 64), "bf16", gpu, 61)
    _check(cache, q, table, [n, 17, 9000], [1, 1, 1], "bf16")
    _check(cache, q * 20, table, [n, 17, 9000], [1, 1, 1], "bf16")


def test_attend_strided_queries(gpu):
    cache, table = _filled(gpu, [70, 33], 2, 128, 16, "bf16", 70)
    fused = _randn((2, 12, 128), "bf16", gpu, 71)
    _check(cache, fused[:, 3:9], table, [70, 33], [1, 1], "bf16")
    other = _randn((6, 2, 128), "bf16", gpu, 72).transpose(0, 1)
    _check(cache, other, table, [70, 33], [1, 1], "bf16")
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    _check(cache, fused[:, 3:9], wide[:, :6], [70, 33], [1, 1], "bf16")


def test_attend_nan_keys_and_values_count_only_where_seen(gpu):
    """NaN in one token of a prompt: queries before it are untouched (also by
    0 * NaN), those after it are NaN: in every channel for a key, in its own
    for a value."""
    dim, n = 64, 100
    cache, table = _filled(gpu, [n], 1, dim, 16, "bf16", 80)
    clean = lm.Cache.of(cache)
    q = _randn((n, 2, dim), "bf16", gpu, 81)
    want, _, bound = lm.attend(clean, _f64(q), table.cpu().numpy(), [n], [n], dim ** -0.5, dtype="bf16")
    off = _i32([0, n], gpu)
    bad = 70
    page = int(table[0, bad // 16])
    v = cache.v.view(torch.uint8)
    keep = v.clone()
    v[page, 0, 0, 5, bad % 16] = 0x7f
    got = _f64(attend_paged_cache(cache, q, table, _i32([n], gpu), offsets=off))
    assert np.isnan(got[bad:, :, 5]).all()
    got[bad:, :, 5] = want[bad:, :, 5]
    assert (np.abs(got - want) <= bound).all()
    windowed = _f64(attend_paged_cache(cache, q, table, _i32([n], gpu), offsets=off, window=10))
    assert np.isnan(windowed[bad:bad + 10, :, 5]).all() and np.isfinite(windowed[bad + 10:]).all()
    v.copy_(keep)
    cache.k.view(torch.uint8)[page, 0, bad % 16, 9] = 0xff
    got = _f64(attend_paged_cache(cache, q, table, _i32([n], gpu), offsets=off))
    assert np.isnan(got[bad:]).all()
    assert (np.abs(got[:bad] - want[:bad]) <= bound[:bad]).all()


def test_attend_bad_indexes_give_nan(gpu):
    cache, table = _filled(gpu, [40, 40, 40], 1, 64, 16, "bf16", 90)
    q = _randn((3, 1, 64), "bf16", gpu, 91)
    bad = table.clone()
    bad[0, 1] = -1
    bad[1, 2] = cache.pages
    out = attend_paged_cache(cache, q, bad, _i32([40, 40, 40], gpu)).cpu()
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2]).all()
    # past the table's width; a negative length holds nothing
    out = attend_paged_cache(cache, q, table, _i32([49, -3, 40], gpu)).cpu()
    assert torch.isnan(out[0]).all() and bool((out[1] == 0).all()) and torch.isfinite(out[2]).all()


def test_attend_queries_that_are_not_finite(gpu):
    cache, table = _filled(gpu, [40, 40], 1, 64, 16, "bf16", 92)
    q = _randn((2, 3, 64), "bf16", gpu, 93)
    want = attend_paged_cache(cache, q, table, _i32([40, 40], gpu))
    q[0, 1, 7] = float("nan")
    got = attend_paged_cache(cache, q, table, _i32([40, 40], gpu))
    assert torch.isnan(got[0, 1]).all()
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)


def test_max_length_is_a_hint(gpu):
    cache, table = _filled(gpu, [3000, 5], 1, 64, 16, "bf16", 94)
    q = _randn((2, 4, 64), "bf16", gpu, 95)
    _check(cache, q, table, [3000, 5], [1, 1], "bf16", max_length=64)


def test_pages_past_32_bits(gpu):
    """Codes more than 2^32 bytes into the cache."""
    pages, heads, dim, page = 70000, 8, 128, 64
    assert pages * heads * dim * page > 1 << 32
    cache = PagedCache.empty(pages, heads, dim, page, gpu)
    rows = [[pages - 1, 0, pages - 2]]
    table = _i32(rows, gpu)
    k, v = (_randn((150, heads, dim), "bf16", gpu, s) for s in (96, 97))
    append_paged_cache(cache, k, v, table, _i32([0], gpu), offsets=_i32([0, 150], gpu))
    q = _randn((1, heads, dim), "bf16", gpu, 98)
    out = attend_paged_cache(cache, q, table, _i32([150], gpu))
    pick = torch.tensor(rows[0], device=gpu)
    small = PagedCache(cache.k.view(torch.uint8)[pick].view(torch.float8_e4m3fn), cache.v.view(torch.uint8)[pick].view(torch.float8_e4m3fn),
                       cache.k_scale[pick], cache.v_scale[pick])
    want = lm.Cache(*(np.zeros((3, heads, page, dim)) for _ in range(2)), *(np.full((3, heads), 2.0 ** -126) for _ in range(2)))
    want.append(_f64(k), _f64(v), [[0, 1, 2]], [0], [150])
    _same(small, want)
    assert torch.equal(out, attend_paged_cache(small, q, _i32([[0, 1, 2]], gpu), _i32([150], gpu)))


def test_empty_calls(gpu):
    cache, table = _filled(gpu, [20], 1, 64, 16, "bf16", 99)
    none = _randn((0, 1, 64), "bf16", gpu, 1)
    zero = _i32([0, 0], gpu)
    assert append_paged_cache(cache, none, none, table, _i32([20], gpu), offsets=zero, q=none).shape == (0, 1, 64)
    assert attend_paged_cache(cache, none, table, _i32([20], gpu), offsets=zero).shape == (0, 1, 64)


def test_side_stream_and_graph(gpu):
    """A decoding step captured once (rotate, append, attend) and replayed on
    new inputs and lengths, every replay equal to the eager step."""
    heads, hq, dim, page = 2, 8, 128, 64
    lengths = [700, 63, 1]
    plan = plan_rotary(dim)
    cache, table = _filled(gpu, [n + 8 for n in lengths], heads, dim, page, "bf16", 110)
    starts, after = _i32(lengths, gpu), _i32([n + 1 for n in lengths], gpu)
    fused = _randn((3, hq + 2 * heads, dim), "bf16", gpu, 111)

    def step():
        q, k, v = fused.split([hq, heads, heads], 1)
        q = append_paged_cache(cache, k, v, table, starts, rotary=plan, q=q)
        return attend_paged_cache(cache, q, table, after)

    want = step()
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        assert torch.equal(step(), want)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for r in range(3):
        fused.copy_(_randn(tuple(fused.shape), "bf16", gpu, 120 + r))
        starts += 1
        after += 1
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step())
    del graph
