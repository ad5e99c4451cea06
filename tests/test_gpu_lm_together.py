"""The operators one after the other, as a serving loop runs them: a prompt with
positions of several axes into shared pages, sequences of their own behind it,
steps of attention over everything and over a window with sinks, a page moved
between caches by reading it back and appending it."""
import numpy as np
import pytest
import torch

import lm_more_oracle as more
import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, RotaryAxes, append_paged_cache, attend_paged_cache, execute_rotary_plan, plan_rotary, read_paged_cache
from test_gpu_paged_cache import _f64, _i32, _randn, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,layout", [("bf16", 128, "half"), ("fp16", 64, "interleaved"), ("bf16", 96, "half")])
def test_a_serving_loop(gpu, dtype, dim, layout):
    print("together", dtype, dim, layout, flush=True)
    heads, hq, page, shared, window, sinks = 2, 8, 16, 5, 40, 6
    tails, steps = [30, 1, 17, 50], 3
    batch, whole = len(tails), shared * page
    pairs = dim // 2
    plan = plan_rotary(dim, layout=layout, axes=RotaryAxes((pairs - 2 * (pairs // 3), pairs // 3, pairs // 3), "cycle"))
    width = -(-(whole + max(tails) + steps) // page)
    order = torch.randperm(shared + batch * (width - shared), generator=torch.Generator().manual_seed(3)).int()
    table = torch.cat([order[:shared].expand(batch, shared), order[shared:].view(batch, -1)], 1).contiguous()
    rows = table.numpy()
    table = table.to(gpu)
    cache = PagedCache.empty(order.numel(), heads, dim, page, gpu)
    want = lm.Cache.of(cache)

    def add(counts, starts, seed):
        """New tokens of the first len(counts) sequences; their turned queries."""
        t = sum(counts)
        q, k, v = _randn((t, hq + 2 * heads, dim), dtype, gpu, seed).split([hq, heads, heads], 1)
        places = torch.randint(0, 5000, (3, t), generator=torch.Generator().manual_seed(seed + 1))
        off = None if counts == [1] * len(counts) else _i32(lm.offsets_of(counts), gpu)
        turned = append_paged_cache(cache, k, v, table[:len(counts)], _i32(starts, gpu), offsets=off, rotary=plan, q=q,
                                    positions=places.to(gpu))
        want.append(more.rotate_axes(_f64(k), places.numpy(), plan), _f64(v), rows, starts, counts)
        y = more.rotate_axes(_f64(q), places.numpy(), plan)
        assert (np.abs(_f64(turned) - y) <= more.rotate_bound(_f64(q), y, dtype, plan)).all()
        assert torch.equal(turned, execute_rotary_plan(plan, q, places.to(gpu)))
        return turned

    def attend(q, lengths, counts):
        """Both kinds of attention over what the cache holds."""
        held = lm.Cache.of(cache)
        off = None if counts == [1] * len(counts) else _i32(lm.offsets_of(counts), gpu)
        got = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, prefix_pages=_i32([shared], gpu))
        y, _, bound = lm.attend(held, _f64(q), rows, lengths, counts, dim ** -0.5, dtype=dtype)
        assert (np.abs(_f64(got) - y) <= bound).all()
        got = attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=off, window=window, sinks=sinks)
        y, _, bound = more.attend(held, _f64(q), rows, lengths, counts, dim ** -0.5, window=window, sinks=sinks, dtype=dtype)
        assert (np.abs(_f64(got) - y) <= bound).all()

    add([whole], [0], 10)
    lengths = [whole + n for n in tails]
    attend(add(tails, [whole] * batch, 20), lengths, tails)
    for s in range(steps):
        q = add([1] * batch, lengths, 30 + 2 * s)
        lengths = [n + 1 for n in lengths]
        attend(q, lengths, [1] * batch)
    _same(cache, want, exact_k=False)

    # everything into a cache of other pages: what is read back is what was
    # cached, and appended again it is the same attention
    total = sum(lengths)
    off = _i32(lm.offsets_of(lengths), gpu)
    k, v = read_paged_cache(cache, table, _i32([0] * batch, gpu), total, offsets=off, dtype=torch.float32)
    held = more.read(lm.Cache.of(cache), rows, [0] * batch, lengths)
    assert (_f64(k) == held[0]).all() and (_f64(v) == held[1]).all()
    size = 64
    wide = -(-max(lengths) // size)
    moved = PagedCache.empty(batch * wide, heads, dim, size, gpu)
    own = torch.arange(batch * wide, dtype=torch.int32, device=gpu).flip(0).view(batch, wide).contiguous()
    append_paged_cache(moved, k, v, own, _i32([0] * batch, gpu), offsets=off)
    out = attend_paged_cache(moved, q, own, _i32(lengths, gpu))
    y, _, bound = lm.attend(lm.Cache.of(moved), _f64(q), own.cpu().numpy(), lengths, [1] * batch, dim ** -0.5, dtype=dtype)
    assert (np.abs(_f64(out) - y) <= bound).all()


def test_a_captured_loop(gpu):
    """Append with positions, both attentions and reading back in one graph,
    replayed as lengths, positions, pages and prefixes change."""
    heads, hq, dim, page, batch, width = 2, 16, 128, 16, 3, 20
    plan = plan_rotary(dim, axes=RotaryAxes((24, 40)))
    caches = [PagedCache.empty(64, heads, dim, page, gpu) for _ in range(2)]
    shared = torch.arange(4, dtype=torch.int32)
    table = torch.cat([shared.expand(batch, 4), torch.arange(4, 4 + batch * (width - 4), dtype=torch.int32).view(batch, -1)], 1).to(gpu)
    starts = [100, 64, 130]
    for cache in caches:
        for row, lo, hi in [(0, 0, 64)] + [(b, 64, n) for b, n in enumerate(starts)]:
            if hi > lo:
                k, v = (_randn((hi - lo, heads, dim), "bf16", gpu, s + row + lo) for s in (1, 2))
                append_paged_cache(cache, k, v, table[row:row + 1], _i32([lo], gpu), offsets=_i32([0, hi - lo], gpu))
    x = _randn((batch, hq + 2 * heads, dim), "bf16", gpu, 50)
    places = torch.zeros((2, batch), dtype=torch.int32, device=gpu)
    lengths, prefix = _i32(starts, gpu), _i32([4], gpu)
    after = lengths + 1

    def step(cache):
        q, k, v = x.split([hq, heads, heads], 1)
        turned = append_paged_cache(cache, k, v, table, lengths, rotary=plan, q=q, positions=places)
        return (attend_paged_cache(cache, turned, table, after, prefix_pages=prefix),
                attend_paged_cache(cache, turned, table, after, window=50, sinks=3),
                *read_paged_cache(cache, table, lengths, batch))

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        for cache in caches:
            step(cache)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = step(caches[0])
    torch.cuda.synchronize()
    for i in range(6):
        x.copy_(_randn((batch, hq + 2 * heads, dim), "bf16", gpu, 60 + i))
        places.copy_(torch.randint(0, 9000, (2, batch), generator=torch.Generator().manual_seed(i)))
        prefix.fill_([4, 0, 2, 3, 4, 1][i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(caches[1])):
            assert torch.equal(a, b)
        lengths += 1
        after += 1
    del graph


def test_two_streams_at_once(gpu):
    """Calls that are cut over the chip, on two streams with nothing to order
    them: each with a workspace of its own, and the same bits as alone."""
    heads, hq, dim, page, batch, shared = 2, 8, 64, 16, 4, 600
    own = 40
    pool = shared + batch * own
    cache = PagedCache.empty(pool, heads, dim, page, gpu)
    every = torch.arange(pool, dtype=torch.int32, device=gpu)
    k, v = (_randn((pool * page, heads, dim), "bf16", gpu, s) for s in (1, 2))
    append_paged_cache(cache, k, v, every[None], _i32([0], gpu), offsets=_i32([0, pool * page], gpu))
    table = torch.cat([every[:shared].expand(batch, shared), every[shared:].view(batch, own)], 1).contiguous()
    q = [_randn((batch, hq, dim), "bf16", gpu, s) for s in (3, 4)]
    lengths = _i32([shared * page + 300 + 90 * b for b in range(batch)], gpu)
    kinds = [dict(prefix_pages=_i32([shared], gpu)), dict(window=7000, sinks=100)]
    alone = [[attend_paged_cache(cache, x, table, lengths, **kw) for kw in kinds] for x in q]
    streams = [torch.cuda.Stream(gpu) for _ in q]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] += [attend_paged_cache(cache, q[i], table, lengths, **kw) for kw in kinds]
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, alone[i][n % 2]) for n, y in enumerate(got[i]))
