"""Attention behind shared pages where the prefix is cut into dozens of parts,
which each sequence's pass adds up: every form of both launches in both types,
groups with rows inside the prefix, with empty and with long rests, large
scores, NaN."""
import pytest
import torch

import lm_device_oracle as dev
import lm_oracle as lm
from kunlunxin_fft_amd import attend_paged_cache, native
from test_gpu_attend_prefix import _shared
from test_gpu_paged_cache import _i32, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture
def workspaces(monkeypatch):
    real, seen = native.cache_attend_with_workspace, []
    monkeypatch.setattr(native, "cache_attend_with_workspace", lambda *a: seen.append(real(*a)) or seen[-1])
    return seen


CASES = [
    # (dim, kv heads, group, page, groups' first sequences, their tokens, tokens behind, counts): by rows a group
    (128, 1, 4, 16, [0, 3], [20000], [700, 1, 9000], [1, 1, 1]),                             # to 16
    (256, 2, 5, 64, [0, 3], [20032], [64, 300, 5], [1, 1, 1]),
    (64, 1, 2, 48, [0, 2, 6], [9600, 20016], [1, 90, 3000, 48, 47, 200], [1] * 6),
    (128, 2, 8, 16, [0, 3], [20000], [700, 1, 9000], [1, 1, 1]),                             # to 32
    (96, 1, 7, 32, [0, 2, 4], [20000, 7008], [33, 900, 1, 2500], [1, 2, 1, 3]),
    (64, 1, 16, 16, [0, 3], [20000], [700, 1, 9000], [1, 1, 1]),                             # to 64
    (96, 2, 12, 16, [0, 4], [20000], [5, 16, 17, 4000], [1, 1, 1, 1]),
    (128, 1, 16, 64, [0, 3], [20032], [700, 1, 9000], [1, 1, 1]),
    (256, 1, 16, 16, [0, 3], [20000], [700, 1, 5000], [1, 1, 1]),                            # head dim 256, many
    (256, 1, 8, 64, [0, 3], [20032], [9, 1, 300], [20, 1, 9]),                               # and rows inside the prefix
    (64, 1, 16, 16, [0, 3], [20000], [9, 700, 5000], [30, 1, 9]),                            # more
    (96, 1, 8, 16, [0, 2, 5], [9008, 20000], [1, 50, 3, 64, 2500], [40, 50, 30, 1, 9]),
    (128, 2, 8, 16, [0, 3], [20000], [700, 1, 9000], [5, 1, 6]),
    (128, 1, 2, 64, [0, 3], [20032], [40, 64, 4000], [100, 1, 60]),
]


def _call(cache, q, table, lengths, counts, cuts, tokens, gpu):
    return attend_paged_cache(cache, q, table, _i32(lengths, gpu), offsets=_i32(lm.offsets_of(counts), gpu), return_lse=True,
                              prefix_pages=_i32([n // cache.page_size for n in tokens], gpu), prefix_groups=_i32(cuts, gpu))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend(gpu, case, dtype, workspaces):
    dim, heads, group, page, cuts, tokens, rests, counts = case
    print("prefix, cut", case, dtype, flush=True)
    assert not any(n % page for n in tokens)
    lengths = [tokens[g] + n for g in range(len(tokens)) for n in rests[cuts[g]:cuts[g + 1]]]
    cache, table = _shared(gpu, cuts, [n // page for n in tokens], lengths, heads, dim, page, dtype, 160, size=2.0)
    for size in (2.0, 30.0):
        q = _randn((sum(counts), heads * group, dim), dtype, gpu, 161, size)
        out, lse = _call(cache, q, table, lengths, counts, cuts, tokens, gpu)
        # more than a row of m, l and O for each row: parts
        assert workspaces[-1] > q.shape[0] * q.shape[1] * (4 * dim + 8) + 2 * 256 * 16 * dim * 4
        dev.check_attend(out, lse, dev.attend(cache, q, table, lengths, counts))
        assert torch.equal(_call(cache, q, table, lengths, counts, cuts, tokens, gpu)[0], out)
    # a place that is free, and a sequence that ends inside the prefix
    short = list(lengths)
    short[0], short[-1] = 0, tokens[-1] - page - 3
    out, lse = _call(cache, q, table, short, counts, cuts, tokens, gpu)
    dev.check_attend(out, lse, dev.attend(cache, q, table, short, counts))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group,count", [(128, 4, 1), (128, 8, 1), (64, 16, 1), (128, 16, 1), (256, 16, 1), (64, 2, 40), (128, 3, 50)], ids=str)
def test_nan_counts_only_where_seen(gpu, dim, group, count, dtype, workspaces):
    """Near the prefix's start, in some part and at its end: every row that sees
    the key; in one's own keys: its own rows."""
    page, prefix, counts = 16, 4000, [count, 1, count]
    lengths = [prefix + 300, prefix + 1, prefix + count // 2 + 1]
    cache, table = _shared(gpu, [0, 3], [prefix // page], lengths, 1, dim, page, dtype, 170)
    q = _randn((sum(counts), group, dim), dtype, gpu, 171)
    want, _, bound = dev.attend(cache, q, table, lengths, counts)
    pos = torch.cat([torch.arange(n - c, n, device=gpu) for n, c in zip(lengths, counts)])
    seq = torch.arange(3, device=gpu).repeat_interleave(torch.tensor(counts, device=gpu))
    v, k = cache.v.view(torch.uint8), cache.k.view(torch.uint8)
    for owner, key in ((None, 7), (None, 2047), (None, prefix - 10), (None, prefix - 1), (0, prefix), (0, lengths[0] - 1)):
        p, slot = int(table[owner or 0, key // page]), key % page
        seen = (pos >= key) & ((seq == owner) if owner is not None else True)
        for codes, at, channel in ((v, (p, 0, 0, 9, slot), 9), (k, (p, 0, slot, 9), slice(None))):
            keep = codes[at].item()
            codes[at] = 0x7f
            got = _call(cache, q, table, lengths, counts, [0, 3], [prefix], gpu)[0].double()
            assert workspaces[-1] > q.shape[0] * q.shape[1] * (4 * dim + 8)
            assert bool(got[seen][..., channel].isnan().all()), key
            hit = torch.zeros_like(got, dtype=torch.bool)
            hit[seen.nonzero()[:, 0][:, None], :, torch.arange(dim, device=gpu)[channel].reshape(1, -1)] = True
            assert bool(((got - want).abs() <= bound)[~hit].all()), key
            codes[at] = keep
