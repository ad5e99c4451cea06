"""Cached tokens read back: every type and layout against codes times scales in
64 bits, ragged starts and lengths, rows of no sequence, bad pages, a graph."""
import numpy as np
import pytest
import torch

import lm_more_oracle as more
import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, native, read_paged_cache
from test_gpu_paged_cache import _f64, _i32, _randn, _table

pytestmark = pytest.mark.gpu


def _random(gpu, pages, heads, dim, page, seed, low=-20, high=8):
    """A cache of every code there is, with scales of many sizes."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(0, 256, (pages, heads, page, dim), generator=g, dtype=torch.uint8).to(gpu)
    v = torch.randint(0, 256, (pages, heads, page // 16, dim, 16), generator=g, dtype=torch.uint8).to(gpu)
    ks, vs = (torch.exp2(torch.randint(low, high, (pages, heads), generator=g).float()).to(gpu) for _ in range(2))
    return PagedCache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs)


def _check(cache, table, starts, counts, dtype, k, v, rows=slice(None)):
    """Codes times powers of two, rounded once to the type: equal bits."""
    with np.errstate(over="ignore"):
        want = torch.from_numpy(more.read(lm.Cache.of(cache), table, starts, counts)).to(lm.DTYPES[dtype])
    for got, w in zip((k, v), want):
        np.testing.assert_array_equal(_f64(got)[rows], _f64(w))


CASES = [
    # (dim, heads, page, starts, counts)
    (128, 1, 16, [0], [1]),
    (128, 8, 64, [0], [77]),
    (64, 3, 16, [5, 0, 16, 31, 47], [1, 1, 1, 1, 1]),
    (96, 2, 32, [0, 7, 33, 15], [100, 25, 1, 17]),
    (256, 1, 48, [3, 40, 0], [40, 0, 48]),
    (128, 4, 128, [100, 0, 127], [300, 16, 2]),
    (64, 16, 16, [9, 0, 31, 17, 4], [0, 33, 0, 15, 600]),
    (96, 5, 1024, [1000, 16], [50, 1008]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_read(gpu, case, dtype):
    dim, heads, page, starts, counts = case
    print("read", case, dtype, flush=True)
    table, pool = _table([a + n for a, n in zip(starts, counts)], page, gpu, 1)
    cache = _random(gpu, pool, heads, dim, page, 2)
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), gpu)
    k, v = read_paged_cache(cache, table, _i32(starts, gpu), sum(counts), offsets=off, dtype=lm.DTYPES[dtype])
    assert k.dtype == v.dtype == lm.DTYPES[dtype] and k.shape == v.shape == (sum(counts), heads, dim)
    _check(cache, table.cpu().numpy(), starts, counts, dtype, k, v)


def test_what_was_appended_comes_back(gpu):
    """Within a code's rounding of it, half a step of three fraction bits, or of
    the least codes of the page."""
    counts, page = [70, 1, 129], 32
    table, pool = _table(counts, page, gpu, 3)
    cache = PagedCache.empty(pool, 2, 128, page, gpu)
    k, v = (_randn((sum(counts), 2, 128), "bf16", gpu, s) for s in (4, 5))
    off = _i32(lm.offsets_of(counts), gpu)
    append_paged_cache(cache, k, v, table, _i32([0, 0, 0], gpu), offsets=off)
    for x, y in zip((k, v), read_paged_cache(cache, table, _i32([0, 0, 0], gpu), sum(counts), offsets=off)):
        top = float(x.abs().max()) / 448 * 2
        assert bool(((x - y).abs().double() <= 2.0 ** -4 * x.abs().double() + 2.0 ** -10 * top).all())
    both = read_paged_cache(cache, table, _i32([60, 0, 64], gpu), 10 + 65, offsets=_i32([0, 10, 10, 75], gpu), dtype=torch.float32)
    whole = read_paged_cache(cache, table, _i32([0, 0, 0], gpu), sum(counts), offsets=off, dtype=torch.float32)
    for part, all_ in zip(both, whole):
        assert torch.equal(part[:10], all_[60:70]) and torch.equal(part[10:], all_[71 + 64:71 + 129])


def test_rows_of_no_sequence_are_zero(gpu):
    table, pool = _table([40, 40], 16, gpu, 6)
    cache = _random(gpu, pool, 3, 64, 16, 7)
    k, v = read_paged_cache(cache, table, _i32([2, 0], gpu), 100, offsets=_i32([5, 43, 70], gpu))
    for t in (k, v):
        assert bool((t[:5] == 0).all()) and bool((t[70:] == 0).all())
    _check(cache, table.cpu().numpy(), [2, 0], [38, 27], "bf16", k, v, slice(5, 70))
    # offsets past the rows: none of them
    k, v = read_paged_cache(cache, table, _i32([0, 0], gpu), 10, offsets=_i32([50, 60, 70], gpu))
    assert bool((k == 0).all()) and bool((v == 0).all())


def test_bad_indexes_give_nan(gpu):
    table, pool = _table([64, 64, 64], 16, gpu, 8)
    cache = _random(gpu, pool, 2, 64, 16, 9)
    bad = table.clone()
    bad[0, 1], bad[1, 0], bad[2, 3] = -1, pool, 1 << 30
    starts, counts = [-3, 0, 40], [30, 70, 30]
    k, v = read_paged_cache(cache, bad, _i32(starts, gpu), 130, offsets=_i32(lm.offsets_of(counts), gpu), dtype=torch.float32)
    _check(cache, bad.cpu().numpy(), starts, counts, "fp32", k, v)
    far = read_paged_cache(cache, bad, _i32([2 ** 31 - 2, -2 ** 31, 2 ** 31 - 1], gpu), 9)
    assert all(bool(torch.isnan(t).all()) for t in far)


def test_scales_past_a_types_range(gpu):
    """float16 cannot hold them all: infinite above, 0 below, as one rounding gives."""
    table, pool = _table([64], 16, gpu, 10)
    cache = _random(gpu, pool, 1, 64, 16, 11, low=-126, high=120)
    for dtype in ("fp16", "bf16", "fp32"):
        k, v = read_paged_cache(cache, table, _i32([0], gpu), 64, dtype=lm.DTYPES[dtype])
        _check(cache, table.cpu().numpy(), [0], [64], dtype, k, v)


def test_strided_tables_and_empty_calls(gpu):
    table, pool = _table([50, 33], 16, gpu, 12)
    cache = _random(gpu, pool, 2, 128, 16, 13)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    k, v = read_paged_cache(cache, wide[:, :5], _i32([1, 1], gpu), 64)
    _check(cache, wide[:, :5].cpu().numpy(), [1, 1], [32, 32], "bf16", k, v)
    k, v = read_paged_cache(cache, table, _i32([0, 0], gpu), 0)
    assert k.shape == v.shape == (0, 2, 128)
    # each its own tensor: what is written to one leaves the other alone
    k, v = read_paged_cache(cache, table, _i32([0, 0], gpu), 2)
    assert k._version == v._version and k.untyped_storage().data_ptr() != v.untyped_storage().data_ptr()


def test_pages_past_32_bits(gpu):
    pages, heads, dim, page = 70000, 8, 128, 64
    assert pages * heads * dim * page > 1 << 32
    cache = PagedCache.empty(pages, heads, dim, page, gpu)
    rows = [[pages - 1, 0, pages - 2]]
    k, v = (_randn((150, heads, dim), "bf16", gpu, s) for s in (96, 97))
    append_paged_cache(cache, k, v, _i32(rows, gpu), _i32([0], gpu), offsets=_i32([0, 150], gpu))
    pick = torch.tensor(rows[0], device=gpu)
    small = PagedCache(cache.k.view(torch.uint8)[pick].view(torch.float8_e4m3fn), cache.v.view(torch.uint8)[pick].view(torch.float8_e4m3fn),
                       cache.k_scale[pick], cache.v_scale[pick])
    k, v = read_paged_cache(cache, _i32(rows, gpu), _i32([0], gpu), 150)
    _check(small, [[0, 1, 2]], [0], [150], "bf16", k, v)


def test_side_stream_and_graph(gpu):
    table, pool = _table([200, 100], 16, gpu, 14)
    cache = _random(gpu, pool, 2, 128, 16, 15)
    starts = _i32([0, 0], gpu)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        read_paged_cache(cache, table, starts, 160)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            k, v = read_paged_cache(cache, table, starts, 160)
    torch.cuda.synchronize()
    for i in range(3):
        starts.copy_(_i32([17 * i, 5 * i], gpu))
        k.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((k, v), read_paged_cache(cache, table, starts, 160)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))  # bits: some are NaN
    del graph


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_outputs_with_strides(gpu, dtype):
    """The C entry's outputs may lie in larger tensors: what is between stays."""
    counts, page, heads, dim = [20, 3, 41], 32, 3, 64
    table, pool = _table([9 + n for n in counts], page, gpu, 11)
    cache = _random(gpu, pool, heads, dim, page, 12)
    t, off, starts = sum(counts), _i32(lm.offsets_of(counts), gpu), _i32([9, 0, 5], gpu)
    fused = torch.full((t, 2 * heads + 1, dim + 16), 7.0, dtype=lm.DTYPES[dtype], device=gpu)
    by_head = torch.full((heads, t + 2, dim), 7.0, dtype=lm.DTYPES[dtype], device=gpu)
    k, v = fused[:, 2:2 + heads, 8:8 + dim], by_head[:, 1:1 + t].transpose(0, 1)
    args = native.READ_ARGS.pack(k.data_ptr(), v.data_ptr(), *k.stride()[:2], *v.stride()[:2], table.data_ptr(), starts.data_ptr(),
                                 off.data_ptr(), table.stride(0), t, table.shape[1], len(counts), getattr(native, dtype.replace("fp", "F").replace("bf", "BF")))
    native.cache_read(cache._packed, args, torch.cuda.current_stream(gpu).cuda_stream)
    for got, want in zip((k, v), read_paged_cache(cache, table, starts, t, offsets=off, dtype=lm.DTYPES[dtype])):
        np.testing.assert_array_equal(_f64(got), _f64(want))
    keep = torch.ones_like(fused, dtype=torch.bool)
    keep[:, 2:2 + heads, 8:8 + dim] = False
    assert bool((fused[keep] == 7).all()) and bool((by_head[:, [0, -1]] == 7).all())
