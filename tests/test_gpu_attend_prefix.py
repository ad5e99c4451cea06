"""Attention of sequences that begin with the same pages: every form of both
launches, groups of any sizes, prefixes that end inside a tile, sequences that
are shorter than their prefix or empty, large scores on either side, NaN."""
import numpy as np
import pytest
import torch

import lm_more_oracle as more
import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, attend_paged_cache
from test_gpu_paged_cache import _f64, _i32, _randn

pytestmark = pytest.mark.gpu


def _shared(gpu, cuts, pages, lengths, heads, dim, page, dtype, seed, size=1.0, spare=3, tail=0):
    """A cache of sequences whose groups share pages, and its table.  What no
    sequence holds is NaN."""
    rng = np.random.default_rng(seed)
    width = max(1, max(-(-n // page) for n in lengths)) + tail
    shared = sum(pages)
    own = []
    for b, n in enumerate(lengths):
        g = [i for i in range(len(pages)) if cuts[i] <= b < cuts[i + 1]]
        own.append(max(0, -(-n // page) - (pages[g[0]] if g else 0)))
    pool = shared + sum(own) + spare
    order = rng.permutation(pool)
    table = np.full((len(lengths), width), -1, np.int32)
    at, holder = shared, {}
    for b, n in enumerate(lengths):
        need = -(-n // page)
        g = [i for i in range(len(pages)) if cuts[i] <= b < cuts[i + 1]]
        p = pages[g[0]] if g else 0
        for i in range(need):
            if i < p:
                table[b, i] = order[sum(pages[:g[0]]) + i]
            else:
                table[b, i] = order[at]
                at += 1
            holder[int(table[b, i])] = True
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    cache.k.view(torch.uint8).fill_(0x7f)
    cache.v.view(torch.uint8).fill_(0xff)
    cache.k_scale.fill_(float("nan"))
    cache.v_scale.fill_(float("nan"))
    used = _i32(sorted(holder), gpu)[:, None]  # each page as a sequence of its own
    if len(holder):
        t = len(holder) * page
        k, v = (_randn((t, heads, dim), dtype, gpu, seed + i, size) for i in (1, 2))
        append_paged_cache(cache, k, v, used, _i32([0] * len(holder), gpu), offsets=_i32(list(range(0, t + 1, page)), gpu))
    return cache, torch.from_numpy(table).to(gpu)


def _check(cache, q, table, lengths, counts, cuts, pages, dtype, want=None, **kw):
    dev = q.device
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), dev)
    out, lse = attend_paged_cache(cache, q, table, _i32(lengths, dev), offsets=off, return_lse=True, prefix_pages=_i32(pages, dev),
                                  prefix_groups=None if cuts is None else _i32(cuts, dev), **kw)
    scale = kw.get("scale") or q.shape[-1] ** -0.5
    want, want_lse, bound = want or lm.attend(lm.Cache.of(cache), _f64(q), table.cpu().numpy(), lengths, counts, scale,
                                              kw.get("causal", True), dtype=dtype)
    got, g = _f64(out), _f64(lse)
    off_by = np.abs(got - want)
    assert (off_by <= bound).all(), f"worst {np.nanmax(off_by / bound)} of the bound, {np.isnan(got).sum()} NaN"
    empty = np.isneginf(want_lse)
    assert (np.isneginf(g) == empty).all() and (got[empty] == 0).all()
    assert (np.abs(g[~empty] - want_lse[~empty]) <= 2.0 ** -16 * (1 + np.abs(want_lse[~empty]))).all()
    return out


CASES = [
    # (dim, kv heads, group, page, groups' first sequences, their pages, lengths, counts, dtype, options)
    (128, 1, 1, 16, [0, 1], [1], [17], [1], "bf16", {}),
    (128, 1, 1, 16, [0, 1], [1], [16], [1], "bf16", {}),
    (128, 2, 4, 64, [0, 6], [3], [193, 200, 300, 192, 256, 700], [1] * 6, "bf16", {}),
    (128, 2, 4, 16, [0, 6], [3], [49, 60, 300, 48, 112, 700], [1] * 6, "fp16", {}),
    (64, 3, 7, 16, [0, 2, 2, 5], [5, 9, 20], [100, 90, 400, 321, 330], [1] * 5, "fp16", {}),
    (96, 1, 16, 32, [0, 3], [7], [225, 400, 0], [1] * 3, "bf16", {}),
    (96, 2, 2, 16, [0, 20], [30], list(range(481, 501)), [1] * 20, "fp16", {}),
    (256, 2, 3, 48, [0, 4], [4], [193, 200, 240, 192], [1] * 4, "fp16", {}),
    (256, 1, 8, 64, [0, 16], [10], [640 + 3 * i for i in range(16)], [1] * 16, "bf16", {}),
    (128, 1, 32, 128, [0, 2], [2], [400, 258], [1] * 2, "bf16", {}),
    (64, 2, 8, 64, [0, 3], [2], [130, 170, 129], [5] * 3, "bf16", {}),
    (128, 2, 2, 16, [0, 2, 5], [4, 2], [100, 140, 70, 0, 66], [33, 1, 5, 2, 40], "fp16", {}),
    (64, 1, 4, 32, [0, 2], [3], [300, 250], [90, 200], "bf16", {}),  # queries inside the prefix
    (128, 2, 4, 32, [0, 3], [20], [700, 813, 640], [60, 300, 640], "bf16", {}),
    (96, 1, 5, 16, [0, 4], [50], [850, 900, 30, 801], [40, 100, 30, 1], "fp16", {}),  # one shorter than the prefix
    (64, 1, 2, 16, [0, 2], [4], [90, 130], [70, 40], "bf16", {"causal": False}),
    (64, 2, 4, 16, [2, 4], [6], [90, 130, 100, 111, 12], [1] * 5, "bf16", {}),  # sequences of no group
    (64, 2, 4, 16, [0, 0, 3, 3], [4, 6, 2], [97, 130, 100], [2] * 3, "fp16", {}),  # groups of none
    (64, 2, 4, 16, [0, 3], [0], [97, 130, 100], [2] * 3, "fp16", {}),  # nothing shared
    (128, 1, 8, 64, [0, 3], [45], [3000, 2881, 2990], [1] * 3, "bf16", {"max_length": 3000}),
    (64, 1, 8, 64, [0, 40], [20], [1281 + i for i in range(40)], [1] * 40, "bf16", {}),
    (128, 4, 7, 16, [0, 9, 24, 70], [40, 3, 17], [641 + 5 * i for i in range(9)] + [49 + i for i in range(15)] + [273 + i for i in range(46)],
     [1] * 70, "bf16", {}),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c)[:90])
def test_attend(gpu, case):
    dim, heads, group, page, cuts, pages, lengths, counts, dtype, kw = case
    print("prefix", case, flush=True)
    cache, table = _shared(gpu, cuts, pages, lengths, heads, dim, page, dtype, 40, size=2.0)
    q = _randn((sum(counts), heads * group, dim), dtype, gpu, 41, 2.0)
    a = _check(cache, q, table, lengths, counts, cuts, pages, dtype, **kw)
    off = None if len(set(counts)) == 1 else _i32(lm.offsets_of(counts), gpu)
    b = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, prefix_pages=_i32(pages, gpu), prefix_groups=_i32(cuts, gpu), **kw)
    assert torch.equal(a, b)  # the same bits every time
    if cuts == [0, len(lengths)]:
        assert torch.equal(_check(cache, q, table, lengths, counts, None, pages, dtype, **kw), a)


@pytest.mark.parametrize("count", [1, 9, 40])
def test_long_prefix(gpu, count):
    """Long enough to be cut over the chip, both parts."""
    lengths = [20000 + 700, 20000 + count, 20000 + 9000]
    cache, table = _shared(gpu, [0, 3], [20000 // 16], lengths, 1, 64, 16, "bf16", 60)
    q = _randn((3 * count, 2, 64), "bf16", gpu, 61)
    _check(cache, q, table, lengths, [count] * 3, [0, 3], [20000 // 16], "bf16")
    _check(cache, q * 20, table, lengths, [count] * 3, [0, 3], [20000 // 16], "bf16")


SIDES = [(1, 1), (1, 24), (3, 16), (5, 16), (70, 4)]


def _with_a_large_key(gpu, key, count, group, dtype):
    """448 in the first channel of a key's codes, 8 in the queries'."""
    lengths, page = [400, 330], 16
    cache, table = _shared(gpu, [0, 2], [16], lengths, 1, 64, page, dtype, 70)
    q = _randn((2 * count, group, 64), dtype, gpu, 71)
    q[..., 0] = 8.0
    for b in range(2):
        cache.k.view(torch.uint8)[int(table[b, key // page]), 0, key % page, 0] = 0x7e
    return cache, table, q, lengths


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("count,group", SIDES)
def test_large_scores(gpu, count, group, dtype):
    """Scores of thousands, the largest in the prefix or after it."""
    for key in (5, 250, 320):
        cache, table, q, lengths = _with_a_large_key(gpu, key, count, group, dtype)
        _check(cache, q, table, lengths, [count] * 2, None, [16], dtype, scale=64.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("count,group", SIDES)
def test_one_key_far_above_the_others(gpu, count, group, dtype):
    """Its page's scale is 64 times larger, so its first channel is 448 * 2^-7
    * 64 = 224 (pages hold values up to 448 * 2^-7 = 3.5 or so), against 8: a
    score of 1792 and 63 products of two normal values, each of the page times
    64.  Where it is the largest by 2 or more, times 64, no other key counts."""
    page = 16
    for key in (5, 250, 320):
        cache, table, q, lengths = _with_a_large_key(gpu, key, count, group, dtype)
        for p in {int(table[b, key // page]) for b in range(2)}:
            cache.k_scale[p] *= 64
        c = lm.Cache.of(cache)
        out = _f64(attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=_i32([0, count, 2 * count], gpu), scale=64.0,
                                      prefix_pages=_i32([16], gpu)))
        some = 0
        for b in range(2):
            k, v = c.tokens(table[b].tolist(), lengths[b])
            for i in range(count):
                pos = lengths[b] - count + i
                s = _f64(q)[b * count + i] @ k[:pos + 1, 0].T
                order = np.sort(s, 1)
                clear = order[:, -1] - order[:, -2] > 2
                some += clear.sum()
                want = v[s.argmax(1), 0]
                u = lm.HALF_ULP[dtype]
                off = np.abs(out[b * count + i] - want)
                assert (off[clear] <= 2 * u * np.abs(want[clear]) + 2.0 ** -20).all(), (key, b, i)
        assert some


@pytest.mark.parametrize("group", [1, 40])
def test_nan_counts_only_where_seen(gpu, group):
    """In the prefix: every row that sees the key, of every sequence; in one's
    own keys: its own rows."""
    lengths, counts, page = [300, 280, 290], [30, 1, 60], 16
    cache, table = _shared(gpu, [0, 3], [15], lengths, 1, 64, page, "bf16", 80)
    q = _randn((sum(counts), group, 64), "bf16", gpu, 81)
    good = lm.attend(lm.Cache.of(cache), _f64(q), table.cpu().numpy(), lengths, counts, 64 ** -0.5)
    want, _, bound = good
    seq = np.repeat(np.arange(3), counts)
    pos = np.concatenate([n - c + np.arange(c) for n, c in zip(lengths, counts)])
    v, k = cache.v.view(torch.uint8), cache.k.view(torch.uint8)
    for owner, key in ((None, 7), (None, 235), (0, 275), (2, 239), (2, 289)):
        p, slot = int(table[owner or 0, key // page]), key % page
        rows = (pos >= key) & (True if key < 240 else seq == owner)
        for bytes_, at, channel in ((v, (p, 0, 0, 9, slot), 9), (k, (p, 0, slot, 9), slice(None))):
            keep = bytes_[at].item()
            bytes_[at] = 0x7f
            got = _f64(attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=_i32(lm.offsets_of(counts), gpu), prefix_pages=_i32([15], gpu)))
            assert np.isnan(got[rows][:, :, channel]).all()
            got[rows, :, channel] = want[rows, :, channel]
            assert (np.abs(got - want) <= bound).all()
            bytes_[at] = keep


def test_an_empty_first_sequence_names_no_pages(gpu):
    """A free place in the batch, whose row of the table is all -1, before and
    between the sequences of the group."""
    lengths, counts = [0, 200, 0, 230], [1] * 4
    cache, table = _shared(gpu, [0, 4], [8], lengths, 2, 128, 16, "bf16", 90)
    assert bool((table[0] == -1).all())
    q = _randn((4, 8, 128), "bf16", gpu, 91)
    _check(cache, q, table, lengths, counts, [0, 4], [8], "bf16")
    lengths = [40, 200, 60, 230]  # and ones that hold a part of it
    table[0, :3] = table[2, :4][:3] = table[1, :3]
    table[2, 3] = table[1, 3]
    _check(cache, q, table, lengths, counts, [0, 4], [8], "bf16")
    _check(cache, q, table, [0, 0, 0, 0], counts, [0, 4], [8], "bf16")


def test_padding_and_bad_indexes(gpu):
    lengths = [200, 230]
    cache, table = _shared(gpu, [0, 2], [8], lengths, 2, 128, 16, "bf16", 95, tail=3)
    q = _randn((7, 8, 128), "bf16", gpu, 96)
    off, pages = _i32([2, 3, 5], gpu), _i32([8], gpu)
    out = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, prefix_pages=pages)
    assert bool((out[[0, 1, 5, 6]] == 0).all())
    want, _, bound = lm.attend(lm.Cache.of(cache), _f64(q)[2:5], table.cpu().numpy(), lengths, [1, 2], 128 ** -0.5)
    assert (np.abs(_f64(out)[2:5] - want) <= bound).all()
    bad = table.clone()
    bad[:, 2] = cache.pages
    out = attend_paged_cache(cache, q, bad, _i32(lengths, gpu), offsets=off, prefix_pages=pages)
    assert torch.isnan(out[2:5]).all() and bool((out[[0, 1, 5, 6]] == 0).all())
    bad = table.clone()
    bad[0, 10] = -1
    out = attend_paged_cache(cache, q, bad, _i32(lengths, gpu), offsets=off, prefix_pages=pages)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[3:5]).all()
    # past the table's width; pages past it, and fewer than none, are those it has, and none
    out = attend_paged_cache(cache, q, table, _i32([10000, 230], gpu), offsets=off, prefix_pages=pages)
    assert torch.isnan(out[2]).all() and torch.isfinite(out[3:5]).all()
    for n, rows in ((1 << 30, slice(3, 5)), (-5, slice(2, 5))):
        cut = table.clone()
        if n > 0:
            cut[0] = table[1]  # all the same then
        out = attend_paged_cache(cache, q, cut, _i32(lengths, gpu), offsets=off, prefix_pages=_i32([n], gpu))
        assert (np.abs(_f64(out)[rows] - want[rows.start - 2:rows.stop - 2]) <= bound[rows.start - 2:rows.stop - 2]).all()
    # groups of sequences that are none: as if they were cut off
    _check(cache, q[:2], table, lengths, [1, 1], [-4, 99], [8], "bf16")


def test_with_a_window_the_prefix_is_not_used(gpu):
    lengths = [200, 230]
    cache, table = _shared(gpu, [0, 2], [8], lengths, 2, 128, 16, "bf16", 97)
    q = _randn((2, 8, 128), "bf16", gpu, 98)
    for kw in (dict(window=60), dict(window=60, sinks=4)):
        a = attend_paged_cache(cache, q, table, _i32(lengths, gpu), **kw)
        assert torch.equal(attend_paged_cache(cache, q, table, _i32(lengths, gpu), prefix_pages=_i32([8], gpu), **kw), a)


def test_two_graphs_and_a_side_stream(gpu):
    """Two captured steps with a workspace each, replayed in turn on lengths
    and shared pages that change between."""
    lengths, dim = [700, 650], 128
    cache, table = _shared(gpu, [0, 2], [40], [n + 200 for n in lengths], 2, dim, 16, "bf16", 100)
    now, pages = _i32(lengths, gpu), _i32([40], gpu)
    qs = [_randn((2, 8, dim), "bf16", gpu, s) for s in (101, 102)]
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in qs], []
    with torch.cuda.stream(side):
        for q, graph in zip(qs, graphs):
            attend_paged_cache(cache, q, table, now, prefix_pages=pages)
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                outs.append(attend_paged_cache(cache, q, table, now, prefix_pages=pages))
    torch.cuda.synchronize()
    for i in range(4):
        now += 37
        pages.fill_((40, 13, 0, 39)[i])
        for q in qs:
            q.copy_(_randn((2, 8, dim), "bf16", gpu, 110 + i))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for q, out in zip(qs, outs):
            assert torch.equal(out, _check(cache, q, table, now.tolist(), [1, 1], None, pages.tolist(), "bf16"))
    del graphs


def test_past_32_bits(gpu):
    """Codes more than 2^32 bytes into the cache, shared and not."""
    pages, heads, dim, page = 70000, 8, 128, 64
    cache = PagedCache.empty(pages, heads, dim, page, gpu)
    rows = [[pages - 1, 0, pages - 2], [pages - 1, 0, 7]]
    x = [_randn((64 * 4, heads, dim), "bf16", gpu, s) for s in (96, 97)]
    append_paged_cache(cache, *x, _i32([[pages - 1], [0], [pages - 2], [7]], gpu), _i32([0] * 4, gpu), offsets=_i32([0, 64, 128, 192, 256], gpu))
    pick = torch.tensor([pages - 1, 0, pages - 2, 7], device=gpu)
    small = PagedCache(cache.k.view(torch.uint8)[pick].view(torch.float8_e4m3fn), cache.v.view(torch.uint8)[pick].view(torch.float8_e4m3fn),
                       cache.k_scale[pick], cache.v_scale[pick])
    q = _randn((2, heads, dim), "bf16", gpu, 98)
    kw = dict(prefix_pages=_i32([2], gpu))
    out = attend_paged_cache(cache, q, _i32(rows, gpu), _i32([150, 190], gpu), **kw)
    assert torch.equal(out, _check(small, q, _i32([[0, 1, 2], [0, 1, 3]], gpu), [150, 190], [1, 1], None, [2], "bf16"))
