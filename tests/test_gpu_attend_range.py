"""Attention over values, weights, scores and page scales of any size, in every
form of the kernel (by the rows a sequence and key head has, and the head dim),
whole and cut over the chip."""
import numpy as np
import pytest
import torch

import lm_oracle as lm
from kunlunxin_fft_amd import PagedCache, append_paged_cache, attend_paged_cache
from test_gpu_paged_cache import _f64, _i32, _randn

pytestmark = pytest.mark.gpu

# (head dim, query heads, queries): 2, 32, 48, 120 rows to head dim 96; 48 and
# 120 rows of 128; 2 and 32 rows of 256
FORMS = [(64, 2, 1), (64, 4, 8), (96, 4, 12), (96, 4, 30), (128, 4, 12), (128, 4, 30), (256, 2, 1), (256, 4, 8)]


def _cache(gpu, k, v, page, spare=1):
    """A cache of one sequence's k and v (tokens, 1, dim) float32, page 0 and
    `spare - 1` others not its; (cache, table)."""
    n, _, dim = k.shape
    need = -(-n // page)
    cache = PagedCache.empty(need + spare, 1, dim, page, gpu)
    table = torch.arange(spare, need + spare, dtype=torch.int32, device=gpu)[None]
    append_paged_cache(cache, k, v, table, _i32([0], gpu), offsets=_i32([0, n], gpu))
    return cache, table


def _attend64(cache, q, table, length, n, window=None):
    """(out, lse, what an element may be off) of one sequence.  Of the sum of
    weighted magnitudes W: the weights' rounding to float16 (2^-11, in
    bfloat16 2^-9 of the 2^-8 allowed), exponentials and sums in 32 bits (2^-18), scores
    accumulated in 32 bits (each, and the maximum, within dim * 2^-24 of the
    sum of magnitudes).  A float16 weight also has a least step, 2^-24 where the
    largest reach 2^13 at least: half of it is 2^-38 of that one, times codes to
    448 of its page, whose scale stands for a magnitude of at least 224: 2^-37
    of the largest magnitude for each key.  Then one rounding of the output."""
    dtype = {torch.float16: "fp16", torch.bfloat16: "bf16"}[q.dtype]
    u, d = lm.HALF_ULP[dtype], q.shape[-1]
    c, x, t = lm.Cache.of(cache), _f64(q), table.cpu().numpy()
    out, lse, _ = lm.attend(c, x, t, [length], [n], d ** -0.5, window=window, dtype=dtype)
    sizes = lm.Cache(np.abs(c.k), np.abs(c.v), c.ks, c.vs)
    weighted, _, _ = lm.attend(lm.Cache(c.k, np.abs(c.v), c.ks, c.vs), x, t, [length], [n], d ** -0.5, window=window, dtype=dtype)
    k, v = sizes.tokens(t[0], length)
    size = (np.abs(x) @ k[:, 0].T).max() * d ** -0.5
    off = weighted * (u + 2.0 ** -18 + 2 * d * 2.0 ** -24 * size)
    if dtype == "fp16":
        off += length * 2.0 ** -37 * v.max()
    return out, lse, off + u * (np.abs(out) + off) + lm.LEAST[dtype]


def _check(got, want, bound):
    off = np.abs(_f64(got) - want)
    assert (off <= bound).all(), f"worst {np.nanmax(off / bound)} of the bound, {np.isnan(off).sum()} NaN"


@pytest.mark.parametrize("length", [180, 3000])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_float16_weights_far_below_the_largest(gpu, dim, heads, n, length):
    """One key 17.5 above the others' scores, with value 0, and thousands with
    value 1: their weights are 2^-25.2 of its own, and count."""
    print("tail", dim, heads, n, length, flush=True)
    k = torch.zeros(length, 1, dim, device=gpu)
    k[3, 0, 0] = 10.0
    v = torch.ones(length, 1, dim, device=gpu)
    v[3] = 0.0
    cache, table = _cache(gpu, k, v, 32)
    q = torch.zeros(n, heads, dim, device=gpu, dtype=torch.float16)
    q[..., 0] = 1.75 * dim ** 0.5
    out, lse = attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu), return_lse=True)
    want, want_lse, bound = _attend64(cache, q, table, length, n)
    assert bound.max() < 0.05 * want.min()
    _check(out, want, bound)
    assert np.abs(_f64(lse) - want_lse).max() <= 2.0 ** -16 * (1 + np.abs(want_lse).max())


@pytest.mark.parametrize("length", [180, 3000])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_float16_queries_over_values_of_any_size(gpu, dim, heads, n, length):
    """Pages of values between 2^-20 and 2^18 in size: no code times its scale
    may overflow while the mean is finite, and rows before a page of large ones
    are untouched."""
    print("values", dim, heads, n, length, flush=True)
    page = 16
    k, v = (_randn((length, 1, dim), "fp32", gpu, s) for s in (300, 301))
    sizes = torch.linspace(-20, 10, -(-length // page), device=gpu).exp2()
    sizes[-2] = 2.0 ** 16
    v *= sizes.repeat_interleave(page)[:length, None, None]
    cache, table = _cache(gpu, k, v, page)
    assert float(cache.v_scale.max()) >= 2.0 ** 9
    q = _randn((n, heads, dim), "fp16", gpu, 302, 0.5)
    out = attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu))
    want, _, bound = _attend64(cache, q, table, length, n)
    assert np.abs(want).max() < 60000
    _check(out, want, bound)


def test_float16_values_that_round_up_past_the_type(gpu):
    """65000 has the code of 65536, which float16 does not hold; their mean with
    the others it does."""
    v = torch.full((40, 1, 64), 65000.0, device=gpu)
    v[::2] = -20000.0
    cache, table = _cache(gpu, torch.zeros(40, 1, 64, device=gpu), v, 16)
    q = _randn((40, 2, 64), "fp16", gpu, 303)
    out = attend_paged_cache(cache, q, table, _i32([40], gpu), offsets=_i32([0, 40], gpu))
    want, _, bound = _attend64(cache, q, table, 40, 40)
    _check(out, want, bound)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 2.0 ** 120])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_pages_before_the_window_may_hold_anything(gpu, dim, heads, n, dtype, scale):
    """Freed pages: entry -1 (which loads read as page 0), or the old number, with
    NaN codes and any scale.  Sixteen-token pages, so that the first group of
    keys the rows share has whole ones before the window."""
    print("window", dim, heads, n, dtype, scale, flush=True)
    length, page, window = 216 if n == 30 else 200, 16, 30
    k, v = (_randn((length, 1, dim), "fp32", gpu, s) for s in (310, 311))
    cache, table = _cache(gpu, k, v, page)
    q = _randn((n, heads, dim), dtype, gpu, 312)
    want, _, bound = _attend64(cache, q, table, length, n, window)
    free = (length - n + 1 - window) // page  # pages no query sees
    assert free % 4  # the last of them share their group with seen ones
    old = [0] + table[0, :free].tolist()
    cache.k.view(torch.uint8)[old] = 0x7f
    cache.v.view(torch.uint8)[old] = 0x7f
    cache.k_scale[old] = scale
    cache.v_scale[old] = scale
    off, lengths = _i32([0, n], gpu), _i32([length], gpu)
    _check(attend_paged_cache(cache, q, table, lengths, offsets=off, window=window), want, bound)
    table[0, :free] = -1
    _check(attend_paged_cache(cache, q, table, lengths, offsets=off, window=window), want, bound)


@pytest.mark.parametrize("length", [150, 3000])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,query", [("bf16", 1e33), ("fp16", 6e4)])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_scores_of_any_size(gpu, dim, heads, n, dtype, query, sign, length):
    """Scores of 2^30 and more, all of one sign: the softmax is the value of the
    largest, alone.  (The weight's own rounding, 2^-11 in float16, is in the
    product and not in the sum.)"""
    print("scores", dim, heads, n, dtype, sign, length, flush=True)
    at = torch.arange(length, device=gpu)
    k = torch.zeros(length, 1, dim, device=gpu)
    size = 1.0 if dtype == "bf16" else 1e6
    k[:, 0, 0] = size * torch.where(at == 5, 1.0 if sign < 0 else 4.0, 2.0 + (at % 3) * 0.25)
    v = _randn((length, 1, dim), "fp32", gpu, 320)
    cache, table = _cache(gpu, k, v, 16)
    q = torch.zeros(n, heads, dim, device=gpu, dtype=lm.DTYPES[dtype])
    q[..., 0] = sign * query
    out, lse = attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu), return_lse=True)
    c = lm.Cache.of(cache)
    ks, vs = c.tokens(table.cpu().numpy()[0], length)
    s = ks[:, 0, 0] * float(q[0, 0, 0]) * dim ** -0.5
    assert s.argmax() == 5 and abs(s[5]) >= 2.0 ** 30
    want = vs[5, 0]
    u = 2.0 ** -11 if dtype == "fp16" else 0.0
    assert (np.abs(_f64(out) - want) <= (u + lm.HALF_ULP[dtype] + 2.0 ** -20) * np.abs(want) + lm.LEAST[dtype]).all()
    assert (np.abs(_f64(lse) - s[5]) <= 2.0 ** -16 * abs(s[5])).all()


@pytest.mark.parametrize("scale", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_a_seen_page_whose_scale_is_none_shows(gpu, dim, heads, n, dtype, scale):
    """Value codes of a page that queries see, under a NaN or infinite scale: NaN
    in every channel, not a number that looks like a result."""
    length = 100
    k, v = (_randn((length, 1, dim), "fp32", gpu, s) for s in (330, 331))
    cache, table = _cache(gpu, k, v, 16)
    cache.v_scale[int(table[0, 1])] = scale
    q = _randn((n, heads, dim), dtype, gpu, 332)
    out = attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu))
    assert not torch.isfinite(out).any()


@pytest.mark.parametrize("length", [160, 2048])
@pytest.mark.parametrize("huge", [-1, 1])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_rows_and_keys_of_very_different_sizes(gpu, dim, heads, n, dtype, huge, length):
    """The first half of the keys score -2^30 or less: what counts is the second
    half, as if alone.  And one query head of scores of 2^30 and more beside the
    others of ordinary ones, which it leaves alone."""
    print("sizes", dim, heads, n, dtype, huge, length, flush=True)
    half, page = length // 2, 16
    k, v = (_randn((length, 1, dim), "fp32", gpu, s) for s in (340, 341))
    k[:, 0, 0] = 0.25
    k[:half] = 0.0
    k[:half, 0, 0] = -1e12 * (1 + torch.arange(half, device=gpu) % 7)
    cache, table = _cache(gpu, k, v, page)
    q = _randn((n, heads, dim), dtype, gpu, 342)
    q[..., 0] = 1.0
    q[:, 1] *= 1e9 if dtype == "bf16" else 1.0
    q[:, 1] = torch.where(torch.isfinite(q[:, 1]), q[:, 1], 0.0)
    if huge < 0:
        q[:, 1] = 0.0
        q[:, 1, 0] = -6e4  # the first half's scores are the large ones here, and positive
    out = _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu)))
    others = [h for h in range(heads) if h != 1]
    want, _, bound = _attend64(cache, q[:, others], table[:, half // page:], half, n)
    assert (np.abs(out[:, others] - want) <= bound).all()
    if huge < 0:  # the value of the first keys of the largest score, alone: seven apart, all equal
        top = lm.Cache.of(cache).tokens(table.cpu().numpy()[0], half)
        s = top[0][:, 0, 0]
        want = top[1][s == s.min(), 0].mean(0)
        size = np.abs(top[1][s == s.min(), 0]).mean(0)
        assert (np.abs(out[:, 1] - want) <= 2 * lm.HALF_ULP[dtype] * size + 2.0 ** -18 * size + lm.HALF_ULP[dtype] * np.abs(want) + lm.LEAST[dtype]).all()
    else:
        assert np.isfinite(out[:, 1]).all()


@pytest.mark.parametrize("length", [160, 2048])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_scores_that_grow_from_small_to_huge(gpu, dim, heads, n, dtype, sign, length):
    """Scores from 2^-20 to 2^36 in the order of the keys, and in the other
    order: the value of the largest that the row sees, alone."""
    print("grow", dim, heads, n, dtype, sign, length, flush=True)
    at = torch.arange(length, device=gpu, dtype=torch.float32)
    k = torch.zeros(length, 1, dim, device=gpu)
    # sixteen keys a page share a scale: a power of two each, within what it holds
    k[:, 0, 0] = torch.exp2(-20 + 56 * torch.floor(at / 16) / (length // 16 - 1)) * (1 + (at % 16) / 16)
    v = _randn((length, 1, dim), "fp32", gpu, 350)
    if sign < 0:
        k, v = k.flip(0), v.flip(0)
    cache, table = _cache(gpu, k, v, 16)
    q = torch.zeros(n, heads, dim, device=gpu, dtype=lm.DTYPES[dtype])
    q[..., 0] = dim ** 0.5
    out = _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu)))
    ks, vs = lm.Cache.of(cache).tokens(table.cpu().numpy()[0], length)
    for i in range(n):
        seen = slice(0, length - n + i + 1)
        s = ks[seen, 0, 0]
        best = s == s.max()
        if s.max() < 2.0 ** 10:
            continue
        want, size = vs[seen][best, 0].mean(0), np.abs(vs[seen][best, 0]).mean(0)
        off = (2 * lm.HALF_ULP[dtype] + 2.0 ** -18) * size + lm.HALF_ULP[dtype] * np.abs(want) + lm.LEAST[dtype]
        assert (np.abs(out[i] - want) <= off).all(), i


@pytest.mark.parametrize("exponent", [0, 19, 20, 21, 24, 25, 26, 27, 40, 90])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_equal_scores_of_any_size(gpu, dim, heads, n, dtype, sign, exponent):
    """Every key scores the same 1.3 * 2^exponent: the mean of the values, whose
    pages are of sizes from 2^-10 to 2^7 (each scale enters the same)."""
    print("equal", dim, heads, n, dtype, sign, exponent, flush=True)
    length, page = 200, 16
    k = torch.zeros(length, 1, dim, device=gpu)
    k[..., 0] = 2.0 ** exponent
    v = _randn((length, 1, dim), "fp32", gpu, 360)
    v *= torch.linspace(-10, 7, -(-length // page), device=gpu).exp2().repeat_interleave(page)[:length, None, None]
    cache, table = _cache(gpu, k, v, page)
    q = torch.zeros(n, heads, dim, device=gpu, dtype=lm.DTYPES[dtype])
    q[..., 0] = sign * 1.3 * dim ** 0.5
    out = _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu)))
    vs = lm.Cache.of(cache).tokens(table.cpu().numpy()[0], length)[1][:, 0]
    for i in range(n):
        want, size = vs[:length - n + i + 1].mean(0), np.abs(vs[:length - n + i + 1]).mean(0)
        off = (lm.HALF_ULP[dtype] + 2.0 ** -18) * size + lm.HALF_ULP[dtype] * np.abs(want) + lm.LEAST[dtype]
        assert (np.abs(out[i] - want) <= off).all(), i


@pytest.mark.parametrize("size", [0.01, 1.0, 40.0, 3000.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,heads,n", FORMS)
def test_a_single_key_gives_its_value(gpu, dim, heads, n, dtype, size):
    """With a window of one, and for a sequence of one key: the value itself, not
    nearly (a weight of one is a power of two, rounded by nothing)."""
    print("single", dim, heads, n, dtype, size, flush=True)
    length, page = 100, 16
    k, v = (_randn((length, 1, dim), "fp32", gpu, s) for s in (370, 371))
    v *= torch.linspace(-6, 6, -(-length // page), device=gpu).exp2().repeat_interleave(page)[:length, None, None]
    cache, table = _cache(gpu, k, v, page)
    q = _randn((n, heads, dim), dtype, gpu, 372, size)
    vs = lm.Cache.of(cache).tokens(table.cpu().numpy()[0], length)[1]
    out = _f64(attend_paged_cache(cache, q, table, _i32([length], gpu), offsets=_i32([0, n], gpu), window=1))
    np.testing.assert_array_equal(out, np.broadcast_to(vs[length - n:], out.shape))
    out = _f64(attend_paged_cache(cache, q[:1], table, _i32([1], gpu), offsets=_i32([0, 1], gpu)))
    np.testing.assert_array_equal(out, np.broadcast_to(vs[:1], out.shape))
