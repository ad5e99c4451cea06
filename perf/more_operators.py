"""More language-model operators whose time is measured, as a user's program
runs them.

* ``rotary``: positions with several axes (time, height, width) rotated into
  query and key heads (``plan_rotary(axes=)``, ``execute_rotary_plan``), with
  the gradient where the case trains;
* ``append``: the same on the way into a paged 8-bit cache, where a token's
  place in the cache is not what it is turned by (``append_paged_cache(
  positions=)``);
* ``read``: cached keys and values read back (``read_paged_cache``);
* ``sinks``: attention in a window whose first tokens stay visible
  (``attend_paged_cache(window=, sinks=)``);
* ``shared``: attention of sequences that begin with the same pages, which are
  read once for all of a group (``attend_paged_cache(prefix_pages=)``).

With ``own`` false the same is computed by elementary torch operations in 32
bits.  Both read the same inputs: a cache is four tensors,

    k        [pages][kv heads][page size][head dim]            float8_e4m3fn
    v        [pages][kv heads][page size / 16][head dim][16]   float8_e4m3fn
    k_scale  [pages][kv heads]                                 float32, 2^e
    v_scale  [pages][kv heads]                                 float32, 2^e

where a page's value is code * scale and e is the least integer for which the
page's largest magnitude is at most 448 * 2^e.

Ranges: 1 to 131072 tokens a call; contexts to 2^18 tokens; 1 to 256 sequences
of mixed lengths, empty ones among them; 1 to 64 query heads over 1 to 16 key
heads; head dims 64, 96, 128 and 256; pages of 16 to 128 tokens; 2 to 4 axes;
1 to 256 sinks; windows to 8192; 1 to 8 shared prefixes.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

MAX_POSITIONS = 1 << 17
BASE = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ----------------------------------------------------------------

def _rotary(batch, seq, heads, dim, axes, order, ladder, layout, dtype, train=False, extra=0, rot=None) -> dict:
    """``extra`` heads lie between one token's heads and the next one's (the
    input is a view of a larger projection)."""
    return {"op": "rotary", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "rot": dim if rot is None else rot,
            "axes": axes, "order": order, "ladder": ladder, "layout": layout, "dtype": dtype, "train": train,
            "extra": extra}


def _append(seqs, new, cached, heads_q, heads_kv, dim, page, dtype, axes=3, order="blocks", ladder="shared",
            layout="half", rot=None) -> dict:
    """``new`` tokens a sequence (1: each exactly one; more: the mean of mixed
    counts) onto up to ``cached`` tokens each."""
    return {"op": "append", "seqs": seqs, "new": new, "cached": cached, "heads_q": heads_q, "heads_kv": heads_kv,
            "dim": dim, "page": page, "dtype": dtype, "axes": axes, "order": order, "ladder": ladder, "layout": layout,
            "rot": dim if rot is None else rot}


def _read(seqs, tokens, first, heads_kv, dim, page, dtype) -> dict:
    """Up to ``tokens`` tokens of each sequence (some none), from a position up
    to ``first`` on; ``first`` 0: exactly as many each, from the start."""
    return {"op": "read", "seqs": seqs, "tokens": tokens, "first": first, "heads_kv": heads_kv, "dim": dim,
            "page": page, "dtype": dtype}


def _sinks(seqs, new, context, window, sinks, heads_q, heads_kv, dim, page, dtype, mixed=False) -> dict:
    """``new`` queries a sequence, the last positions of contexts of up to
    ``context`` tokens (``mixed``: of any length up to it, some empty)."""
    return {"op": "sinks", "seqs": seqs, "new": new, "context": context, "window": window, "sinks": sinks,
            "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim, "page": page, "dtype": dtype, "mixed": mixed}


def _shared(seqs, groups, prefix, rest, new, heads_q, heads_kv, dim, page, dtype, mixed=False) -> dict:
    """``seqs`` sequences in ``groups`` groups, each group's with the same first
    ``prefix`` tokens (whole pages of them; ``mixed``: up to it) and up to
    ``rest`` tokens of their own, of which the last ``new`` are the queries."""
    return {"op": "shared", "seqs": seqs, "groups": groups, "prefix": prefix, "rest": rest, "new": new,
            "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim, "page": page, "dtype": dtype, "mixed": mixed}


def listed() -> list:
    return [
        # the query and key heads of one token, a view of its fused projection: one step of a reply about a picture
        {"name": "axes_token", **_rotary(1, 1, 40, 128, 3, "blocks", "shared", "half", "bf16", extra=8)},
        # a training batch of text and pictures, forward and gradient
        {"name": "axes_train", **_rotary(2, 4096, 32, 128, 3, "blocks", "shared", "half", "bf16", train=True)},
        # the patches of a video, an odd number, in 32 bits, each axis with frequencies of its own, neighbouring pairs
        {"name": "axes_patches", **_rotary(1, 50001, 16, 64, 3, "cycle", "own", "interleaved", "fp32", train=True)},
        # prompts of text and pictures written to the cache, keys and queries rotated
        {"name": "append_axes", **_append(4, 4096, 1000, 32, 8, 128, 64, "bf16")},
        # a short sequence taken out of the cache: latency
        {"name": "read_short", **_read(1, 77, 0, 8, 128, 64, "bf16")},
        # a batch of mixed lengths and starts, some empty, short pages
        {"name": "read_mixed", **_read(64, 4096, 3000, 4, 128, 16, "fp16")},
        # one very long context: bandwidth
        {"name": "read_long", **_read(1, 1 << 17, 0, 8, 128, 64, "bf16")},
        # one token of an endless reply: latency
        {"name": "sinks_token", **_sinks(1, 1, 20000, 1024, 4, 32, 8, 128, 64, "bf16")},
        # a serving batch of mixed lengths, seven query heads a key head, short pages
        {"name": "sinks_batch", **_sinks(64, 1, 16384, 4096, 16, 28, 4, 128, 16, "fp16", mixed=True)},
        # a piece of a long prompt in its window: matrix products
        {"name": "sinks_chunk", **_sinks(1, 2048, 32768, 4096, 128, 32, 8, 128, 64, "bf16")},
        # many replies under one long instruction, one token each
        {"name": "shared_decode", **_shared(64, 1, 32768, 1000, 1, 32, 8, 128, 64, "bf16")},
        # questions about a few documents, a piece of a prompt each
        {"name": "shared_prompts", **_shared(32, 3, 16384, 700, 64, 28, 4, 128, 16, "fp16", mixed=True)},
    ]


def _log(rng, low, high) -> int:
    return max(low, min(high, int(2.0 ** rng.uniform(math.log2(low), math.log2(high + 1)))))


def _cost(case) -> float:
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng) -> dict:
    while True:
        case = _drawn(rng)
        if _cost(case) <= max(map(_cost, listed())):
            return case


def _drawn(rng) -> dict:
    op = rng.choice(["rotary", "rotary", "append", "read", "sinks", "sinks", "shared", "shared"])
    dim = rng.choice([64, 96, 128, 128, 256])
    turn = {"axes": rng.choice([2, 3, 3, 4]), "order": rng.choice(["blocks", "cycle"]),
            "ladder": rng.choice(["shared", "own"]), "layout": rng.choice(["half", "interleaved"]),
            "rot": rng.choice([dim, dim, dim // 2, 20])}
    if op == "rotary":
        batch, heads = _log(rng, 1, 64), rng.randint(1, 64)
        # at most 2^28 values
        seq = _log(rng, 1, max(1, min(131072, (1 << 28) // (batch * heads * dim))))
        return _rotary(batch, seq, heads, dim, dtype=rng.choice(["bf16", "fp16", "fp32"]), train=rng.random() < 0.5,
                       extra=rng.choice([0, 0, 8]), **turn)
    heads_kv = rng.choice([1, 2, 4, 8, 16])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 7, 8] if heads_kv <= 8 else [1, 2, 4])
    page, dtype, seqs = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "fp16"]), _log(rng, 1, 256)
    if op == "append":
        # at most 2^27 values of q
        most = max(1, min(8192, (1 << 27) // (seqs * heads_q * dim)))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, most)
        return _append(seqs, new, _log(rng, 1, 8192), heads_q, heads_kv, dim, page, rng.choice(["bf16", "fp16", "fp32"]),
                       **turn)
    if op == "read":
        # at most 2^28 codes
        most = max(1, min(1 << 18, (1 << 27) // (seqs * heads_kv * dim)))
        return _read(seqs, _log(rng, 1, most), rng.choice([0, _log(rng, 1, 4096)]), heads_kv, dim, page,
                     rng.choice(["bf16", "fp16", "fp32"]))
    new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 1024)])
    if op == "sinks":
        # at most 2^29 bytes of cache and 2^38 operations a product
        most = min(1 << 18, (1 << 28) // (seqs * heads_kv * dim), (1 << 37) // (seqs * new * heads_q * dim))
        context = _log(rng, 1, max(1, most))
        return _sinks(seqs, min(new, context), context, _log(rng, 1, 8192), _log(rng, 1, 256), heads_q, heads_kv, dim,
                      page, dtype, rng.random() < 0.5)
    groups = rng.randint(1, min(8, seqs))
    rest = new + _log(rng, 1, 2000)
    # at most 2^29 bytes of cache, 2^38 operations a product, and 2^24 keys that the sequences have together
    most = min(1 << 17, (1 << 28) // (groups * heads_kv * dim), (1 << 37) // (seqs * new * heads_q * dim),
               (1 << 34) // (seqs * heads_kv * dim))
    return _shared(seqs, groups, _log(rng, 1, max(1, most)), rest, new, heads_q, heads_kv, dim, page, dtype,
                   rng.random() < 0.5)


# ---- sizes a case fixes ---------------------------------------------------

def _fixed(case):
    """Random numbers that follow from the case alone, so that every seed's
    inputs are the same work."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _groups(case):
    """(sequences before each group and after the last, pages that each group shares)."""
    r, n, g = _fixed(case), case["seqs"], case["groups"]
    cuts = [0, *sorted(r.randint(0, n) for _ in range(g - 1)), n] if case["mixed"] else [n * i // g for i in range(g + 1)]
    return cuts, [(r.randint(0, case["prefix"]) if case["mixed"] and i else case["prefix"]) // case["page"]
                  for i in range(g)]


def _lengths(case):
    """(new tokens, tokens in the cache) of each sequence: before the new ones
    for ``append`` and ``read``, with them for attention."""
    r, n, op = _fixed(case), case["seqs"], case["op"]
    if op == "append":
        new = [1 if case["new"] == 1 else r.randint(1, 2 * case["new"] - 1) for _ in range(n)]
        return new, [r.randint(0, case["cached"]) for _ in range(n)]
    if op == "read":
        if not case["first"]:
            return [case["tokens"]] * n, [0] * n
        return ([case["tokens"]] + [0 if r.random() < 0.1 else r.randint(1, case["tokens"]) for _ in range(n - 1)],
                [r.randint(0, case["first"]) for _ in range(n)])
    new = [case["new"]] * n
    if op == "shared":
        cuts, pages = _groups(case)
        full = []
        for i, p in enumerate(pages):
            for _ in range(cuts[i], cuts[i + 1]):
                full.append(p * case["page"] + r.randint(case["new"], case["rest"]))
        if case["mixed"]:  # an empty place in the batch
            full = [0 if r.random() < 0.05 else x for x in full]
            if case["new"] > 1:
                new = [min(r.randint(1, case["new"]), x) if x else 1 for x in full]
        return new, full
    full = [case["context"]] * n
    if case["mixed"]:
        full = [r.choice([0, case["context"]]) if r.random() < 0.1 else r.randint(1, case["context"]) for _ in range(n)]
        if case["new"] > 1:
            new = [r.randint(0, case["new"]) for _ in range(n)]
        full[0], new[0] = case["context"], case["new"]
    return new, full


def _pairs(case):
    """How many pairs each axis turns: time fewer than the others."""
    n, axes = case["rot"] // 2, case["axes"]
    out = [n // 4 if axes == 3 else n // axes]
    while len(out) < axes:
        out.append((n - sum(out)) // (axes - len(out)))
    return out


def _axis_of(case):
    """(axis, place among the axis' own pairs) of each pair."""
    left, place, out = _pairs(case), [0] * case["axes"], []
    while sum(left):
        for a in range(case["axes"]):
            for _ in range(left[a] if case["order"] == "blocks" else min(1, left[a])):
                out.append((a, place[a]))
                place[a] += 1
                left[a] -= 1
    return out


def _frequencies(case):
    """Radians a position of each pair, in 64 bits."""
    n = _pairs(case)
    return [BASE ** (-2.0 * (i / (2 * n[a]) if case["ladder"] == "own" else j / case["rot"]))
            for j, (a, i) in enumerate(_axis_of(case))]


@functools.lru_cache(maxsize=4)
def _table(freqs, device):
    """cos and sin of every position, made in 64 bits: what a program without
    this library keeps beside the model."""
    a = torch.arange(MAX_POSITIONS, device=device, dtype=torch.float64)[:, None] * torch.tensor(
        freqs, device=device, dtype=torch.float64)
    return a.cos().float(), a.sin().float()


# ---- inputs ---------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _places(rng, case, tokens):
    """Positions (axes, tokens) of one sequence of text and pictures: a text's
    tokens go on along all axes alike, a picture's along the last two (a
    film's along the last three); what follows goes on past the largest."""
    axes, parts, at, have = case["axes"], [], rng.randint(0, 1000), 0
    while have < tokens:
        if rng.random() < 0.5:
            n = rng.randint(1, 400)
            parts.append((at + torch.arange(n)).expand(axes, n))
            at += n
        else:
            shape = [rng.randint(1, 4) for _ in range(axes - 2)] + [rng.randint(4, 40), rng.randint(4, 40)]
            parts.append(at + torch.stack([g.reshape(-1) for g in torch.meshgrid(
                *(torch.arange(s) for s in shape), indexing="ij")]))
            at += max(shape)
        have += parts[-1].shape[1]
    return torch.cat(parts, 1)[:, :tokens]


def _block_exponent(amax):
    """The least e with amax <= 448 * 2^e (448 = 0.875 * 2^9), at least -126."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (m > 0.875).int(), torch.full_like(x, -126)).clamp(-126, 120)


def _two_to(e):
    return torch.ldexp(torch.ones((), device=e.device), e)


def _random_pages(g, pages, heads, shape):
    """Codes and scales of pages full of N(0, 1) values, each page and head
    with a size of its own."""
    dev = _device()
    codes = torch.empty((pages, heads) + shape, device=dev, dtype=torch.float8_e4m3fn)
    scale = torch.empty((pages, heads), device=dev)
    step = max(1, (1 << 26) // (heads * math.prod(shape)))
    dims = tuple(range(2, 2 + len(shape)))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        x = torch.randn((n, heads) + shape, generator=g, device=dev)
        x *= torch.empty((n, heads) + (1,) * len(shape), device=dev).uniform_(0.7, 1.4, generator=g)
        s = _two_to(_block_exponent(x.abs().amax(dims)))
        scale[a:a + n] = s
        codes[a:a + n] = (x / s.reshape((n, heads) + (1,) * len(shape))).to(torch.float8_e4m3fn)
    return codes, scale


def _paged(g, case, full):
    """The cache tensors and the page table of sequences of ``full`` tokens:
    pages anywhere in the pool, unused entries -1; a group's first pages are
    the same for all its sequences."""
    dev, size = _device(), case["page"]
    need = [-(-n // size) for n in full]
    group, first = [], []  # of each sequence: its group, and its pages before its own
    if case["op"] == "shared":
        cuts, pages = _groups(case)
        for i, p in enumerate(pages):
            group += [i] * (cuts[i + 1] - cuts[i])
        first = [min(pages[i], n) for i, n in zip(group, need)]
        base = [sum(pages[:i]) for i in range(len(pages))]
        shared = sum(pages)
    else:
        group, first, base, shared = [0] * len(need), [0] * len(need), [0], 0
    pool = shared + sum(need) - sum(first) + 3
    k, ks = _random_pages(g, pool, case["heads_kv"], (size, case["dim"]))
    v, vs = _random_pages(g, pool, case["heads_kv"], (size // 16, case["dim"], 16))
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    width = max(1, max(need))
    count, same = torch.tensor(need, device=dev), torch.tensor(first, device=dev)
    at = torch.arange(width, device=dev)[None]
    mine = shared + torch.cumsum(count - same, 0) - (count - same)
    place = torch.where(at < same[:, None], torch.tensor([base[i] for i in group], device=dev)[:, None] + at,
                        mine[:, None] + at - same[:, None])
    table = order[place.clamp(max=pool - 1)]
    table = torch.where(at < count[:, None], table, torch.full_like(table, -1))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "page_table": table.contiguous()}


def _offsets(new):
    c = [0]
    for n in new:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=_device())


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=_device())


def prepare(case: dict, seed: int) -> dict:
    dev = _device()
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rng = random.Random(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev).to(dt)

    s = {"case": case}
    if op == "rotary":
        b, n, h, d = case["batch"], case["seq"], case["heads"], case["dim"]
        s["x"] = randn(b, n, h + case["extra"], d)[:, :, :h]
        s["positions"] = torch.stack([_places(rng, case, n) for _ in range(b)], 1).to(dev)
        if case["train"]:
            s["x"].requires_grad_()
            s["grad"] = randn(b, n, h, d)
        s["roots"] = _table(tuple(_frequencies(case)), dev)
        return s
    new, full = _lengths(case)
    t = sum(new)
    if op == "append":
        s |= _paged(g, case, [a + b for a, b in zip(new, full)])
        fused = randn(t, case["heads_q"] + 2 * case["heads_kv"], case["dim"])  # one projection's output
        s["q"], s["new_k"], s["new_v"] = fused.split([case["heads_q"], case["heads_kv"], case["heads_kv"]], dim=1)
        s["starts"] = _int32(full)
        s["positions"] = torch.cat([_places(rng, case, n) for n in new], 1).to(dev)
        s["roots"] = _table(tuple(_frequencies(case)), dev)
    elif op == "read":
        s |= _paged(g, case, [a + b for a, b in zip(new, full)])
        s["starts"], s["tokens"] = _int32(full), t
    else:
        s |= _paged(g, case, full)
        s["q"] = randn(t, case["heads_q"], case["dim"])
        s["lengths"] = _int32(full)
        s["max_length"], s["max_new"] = max(full), max(new)
        if op == "shared":
            cuts, pages = _groups(case)
            s["prefix_groups"], s["prefix_pages"] = _int32(cuts), _int32(pages)
    even = case["new"] if op in ("sinks", "shared") else case["tokens"] if op == "read" and not case["first"] else 1
    s["offsets"] = None if all(n == even for n in new) else _offsets(new)
    return s


# ---- one pass -------------------------------------------------------------

def _rotated(x, cos, sin, layout):
    """x [..., dim] with its first 2 * pairs channels rotated; 32 bits."""
    p = cos.shape[-1]
    x = x.float()
    if layout == "half":
        a, b, rest = x[..., :p], x[..., p:2 * p], x[..., 2 * p:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b, rest = x[..., 0:2 * p:2], x[..., 1:2 * p:2], x[..., 2 * p:]
    y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _roots_of(s):
    """cos and sin [..., 1, pairs] of the positions [axes, ...]."""
    axis = [a for a, _ in _axis_of(s["case"])]
    at = s["positions"].movedim(0, -1)[..., axis]  # [..., pairs]
    pair = torch.arange(len(axis), device=at.device)
    return (t[at, pair].unsqueeze(-2) for t in s["roots"])


def _plain_rotary(s):
    c, x = s["case"], s["x"].detach()
    cos, sin = _roots_of(s)
    y = _rotated(x, cos, sin, c["layout"]).to(x.dtype)
    if not c["train"]:
        return {"y": y}
    return {"y": y, "x_grad": _rotated(s["grad"], cos, -sin, c["layout"]).to(x.dtype)}


def _sequence_of(offsets, tokens, sequences):
    """Which sequence each token belongs to, and its place in it."""
    at = torch.arange(tokens, device=_device())
    if offsets is None:
        per = tokens // sequences
        return at // per, at % per
    seq = torch.searchsorted(offsets[1:], at, right=True)
    return seq, at - offsets[seq]


def _plain_append(s):
    c, k, v = s["case"], s["new_k"], s["new_v"]
    size, t = c["page"], k.shape[0]
    starts = s["starts"].long()
    seq, place = _sequence_of(s["offsets"], t, starts.numel())
    pos = starts[seq] + place
    cos, sin = _roots_of(s)
    q = _rotated(s["q"], cos, sin, c["layout"]).to(s["q"].dtype)
    page, slot = s["page_table"][seq, pos // size].long(), pos % size
    # the page each sequence goes on filling, and whether it holds anything yet
    going = s["page_table"][torch.arange(starts.numel(), device=k.device), starts // size].long()
    held = starts % size
    for x, codes, scale, is_v in ((_rotated(k, cos, sin, c["layout"]), s["k"], s["k_scale"], False),
                                  (v.float(), s["v"], s["v_scale"], True)):
        peak = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
        kept = torch.where(held[:, None] > 0, scale[going], torch.zeros((), device=k.device))
        now = _two_to(_block_exponent(peak))
        grown = torch.maximum(now[going], kept)
        shrink = torch.where(held[:, None] > 0, kept / grown, torch.ones((), device=k.device))
        old = codes[going].float()
        shrink = shrink.reshape(shrink.shape + (1,) * (old.dim() - 2))
        codes[going] = (old * shrink).to(codes.dtype)
        scale[page] = now[page]
        scale[going] = grown
        y = (x / scale[page][..., None]).to(codes.dtype)
        if is_v:
            codes[page, :, slot // 16, :, slot % 16] = y
        else:
            codes[page, :, slot] = y
    return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_read(s):
    c, size = s["case"], s["case"]["page"]
    seq, place = _sequence_of(s["offsets"], s["tokens"], c["seqs"])
    pos = s["starts"].long()[seq] + place
    page, slot = s["page_table"][seq, pos // size].long(), pos % size
    # (indexed in 8 bits, as raw bytes: indexing converts nothing)
    k = s["k"].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn)
    v = s["v"].view(torch.uint8)[page, :, slot // 16, :, slot % 16].contiguous().view(torch.float8_e4m3fn)
    dt = DTYPES[c["dtype"]]
    return {"k": (k.float() * s["k_scale"][page][..., None]).to(dt), "v": (v.float() * s["v_scale"][page][..., None]).to(dt)}


def _plain_attend(s):
    """All keys of a sequence, masked; a few sequences at a time where all would not fit."""
    c, q = s["case"], s["q"]
    size, dim, hk = c["page"], c["dim"], c["heads_kv"]
    group, n, t = c["heads_q"] // hk, s["max_new"], q.shape[0]
    total, width = s["page_table"].shape
    length = width * size
    seq, place = _sequence_of(s["offsets"], t, total)
    count = torch.full((total,), t // total, device=q.device) if s["offsets"] is None else s["offsets"].diff().long()
    padded = torch.zeros(total, n, hk, group, dim, device=q.device)
    padded[seq, place] = q.float().reshape(t, hk, group, dim)
    result = torch.empty_like(padded)
    step = max(1, (1 << 32) // (length * hk * (2 * dim + 2 * n * group)))
    for i in range(0, total, step):
        pages = s["page_table"][i:i + step].clamp(min=0).long()
        b = pages.shape[0]
        k = s["k"][pages].float() * s["k_scale"][pages][..., None, None]
        k = k.transpose(1, 2).reshape(b, hk, length, dim)
        v = s["v"][pages].float() * s["v_scale"][pages][..., None, None, None]
        v = v.permute(0, 2, 1, 3, 5, 4).reshape(b, hk, length, dim)
        rows = padded[i:i + step].permute(0, 2, 1, 3, 4).reshape(b, hk, n * group, dim)
        score = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * dim ** -0.5
        at = torch.arange(length, device=q.device)
        pos = (s["lengths"][i:i + step] - count[i:i + step])[:, None] + torch.arange(n, device=q.device)  # [b][n]
        seen = at <= pos[..., None]
        if c["op"] == "sinks":
            seen &= (at > pos[..., None] - c["window"]) | (at < c["sinks"])
        seen = seen[:, None, :, None].expand(b, 1, n, group, length).reshape(b, 1, n * group, length)
        score = score.masked_fill_(~seen, -math.inf)
        top = score.amax(-1, keepdim=True)
        p = (score - top.masked_fill(top == -math.inf, 0.0)).exp_()
        sums = p.sum(-1, keepdim=True)
        out = torch.matmul(p, v) / sums.masked_fill(sums == 0, 1.0)
        result[i:i + step] = out.reshape(b, hk, n, group, dim).permute(0, 2, 1, 3, 4)
    return {"out": result[seq, place].reshape(t, c["heads_q"], dim).to(q.dtype)}


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own_pass(s):
    pkg, c, op = _package(), s["case"], s["case"]["op"]
    if "handles" not in s:  # what a program keeps beside its tensors
        s["handles"] = True
        if op in ("rotary", "append"):
            s["plan"] = pkg.plan_rotary(c["dim"], rot_dim=c["rot"], layout=c["layout"], base=BASE,
                                        axes=pkg.RotaryAxes(tuple(_pairs(c)), c["order"], c["ladder"]),
                                        max_positions=MAX_POSITIONS)
        if op != "rotary":
            s["cache"] = pkg.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if op == "rotary":
        y = pkg.execute_rotary_plan(s["plan"], s["x"], s["positions"])
        if not c["train"]:
            return {"y": y}
        return {"y": y.detach(), "x_grad": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    if op == "append":
        q = pkg.append_paged_cache(s["cache"], s["new_k"], s["new_v"], s["page_table"], s["starts"],
                                   offsets=s["offsets"], rotary=s["plan"], positions=s["positions"], q=s["q"])
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if op == "read":
        k, v = pkg.read_paged_cache(s["cache"], s["page_table"], s["starts"], s["tokens"], offsets=s["offsets"],
                                    dtype=DTYPES[c["dtype"]])
        return {"k": k, "v": v}
    more = ({"window": c["window"], "sinks": c["sinks"]} if op == "sinks" else
            {"prefix_pages": s["prefix_pages"], "prefix_groups": s["prefix_groups"]})
    return {"out": pkg.attend_paged_cache(s["cache"], s["q"], s["page_table"], s["lengths"], offsets=s["offsets"],
                                          max_length=s["max_length"], **more)}


def run(state: dict):
    if own:
        return _own_pass(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "read": _plain_read, "sinks": _plain_attend,
            "shared": _plain_attend}[state["case"]["op"]](state)


def _seen(case):
    """(keys to read, query and key pairs) of an attention over all sequences:
    what any query of a sequence sees, a shared prefix once a group."""
    keys = pairs = 0
    new, full = _lengths(case)
    for n, length in zip(new, full):
        first = max(0, length - n)  # position of the first query that sees anything
        if length <= first:
            continue
        every = length * (length + 1) // 2 - first * (first + 1) // 2
        if case["op"] == "sinks":
            w, s = case["window"], case["sinks"]
            low = max(0, first - w + 1)
            keys += length - low + min(s, low)
            # a query at p misses those from s to p - w, of p + 1
            for p in range(max(first, w + s), length):
                every -= p - w + 1 - s
        else:
            keys += length
        pairs += every
    if case["op"] == "shared":
        cuts, pages = _groups(case)
        for i, p in enumerate(pages):
            there = sum(1 for x in full[cuts[i]:cuts[i + 1]] if x)
            keys -= max(0, there - 1) * p * case["page"]
    return keys, pairs


def work(case: dict) -> dict:
    """Each input read once, each output written once: the rotated heads and
    their gradient (6 operations a pair) and the positions; the new keys,
    values and queries and their codes; the codes read back (one product
    each); the visible codes with their scales, the queries and outputs (two
    products of ``dim`` for a query head and key that see each other)."""
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * tokens * (2 * case["heads"] * case["dim"] * size + 8 * case["axes"]),
                "flops": passes * tokens * case["heads"] * 3 * case["rot"]}
    kv = 2 * case["heads_kv"] * case["dim"]
    t = sum(_lengths(case)[0])
    if case["op"] == "append":
        return {"bytes": t * (kv * (size + 1) + 2 * case["heads_q"] * case["dim"] * size + 8 * case["axes"]),
                "flops": t * (3 * (case["heads_q"] + case["heads_kv"]) * case["rot"] + 2 * kv)}
    if case["op"] == "read":
        return {"bytes": t * (kv * (size + 1) + 8.0 * case["heads_kv"] / case["page"]), "flops": t * kv}
    keys, pairs = _seen(case)
    return {"bytes": keys * case["heads_kv"] * (2 * case["dim"] + 8.0 / case["page"])
            + 2 * t * case["heads_q"] * case["dim"] * size,
            "flops": 4 * pairs * case["heads_q"] * case["dim"]}


# ---- in 64 bits -----------------------------------------------------------

def _turn64(x, pos, case, sign=1):
    """x [tokens, heads, dim] as complex pairs times exp(i pos theta); pos [axes, tokens]."""
    p = case["rot"] // 2
    angle = torch.empty(x.shape[0], p, device=x.device, dtype=torch.float64)
    for j, ((a, _), f) in enumerate(zip(_axis_of(case), _frequencies(case))):
        angle[:, j] = sign * pos[a].double() * f
    root = torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.double().clone()
    one, two = (slice(0, p), slice(p, 2 * p)) if case["layout"] == "half" else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    z = torch.complex(y[..., one].contiguous(), y[..., two].contiguous()) * root
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _round_e4m3(x):
    """The nearest value with 3 fraction bits and an exponent of at least -6, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        b, n, h, d = s["x"].shape
        pos = s["positions"].reshape(case["axes"], -1)
        out = {"y": _turn64(s["x"].detach().reshape(-1, h, d), pos, case).reshape(b, n, h, d)}
        if case["train"]:
            out["x_grad"] = _turn64(s["grad"].reshape(-1, h, d), pos, case, -1).reshape(b, n, h, d)
        return out
    new, full = _lengths(case)
    size, dev = case["page"], _device()
    if case["op"] == "append":
        k, v = _turn64(s["new_k"], s["positions"], case), s["new_v"].double()
        ck, cv = s["k"].double(), s["v"].double()
        sk, sv = s["k_scale"].double(), s["v_scale"].double()
        at, table = 0, s["page_table"].tolist()
        for i, (n, a) in enumerate(zip(new, full)):
            p = a
            while p < a + n:  # one page at a time
                m = min(size - p % size, a + n - p)
                page, o = table[i][p // size], p % size
                for x, codes, scale in ((k, ck, sk), (v, cv, sv)):
                    new_x = x[at:at + m].transpose(0, 1)  # [heads][m][dim]
                    mant, e = torch.frexp(new_x.abs().amax((1, 2)))
                    e = torch.where(mant > 0, e.double() - torch.where(mant > 0.875, 8.0, 9.0), -126.0).clamp(-126, 120)
                    was = scale[page].clone()
                    if o:
                        scale[page] = torch.maximum(was, torch.exp2(e))
                        codes[page] = _round_e4m3(codes[page] * (was / scale[page]).reshape(
                            (-1,) + (1,) * (codes.dim() - 2)))
                    else:
                        scale[page] = torch.exp2(e)
                    y = _round_e4m3(new_x / scale[page][:, None, None])
                    if codes is ck:
                        codes[page][:, o:o + m] = y
                    else:
                        slot = torch.arange(o, o + m, device=y.device)
                        codes[page][:, slot // 16, :, slot % 16] = y.transpose(0, 1)
                p, at = p + m, at + m
        return {"q": _turn64(s["q"], s["positions"], case), "k": ck, "v": cv, "k_scale": sk, "v_scale": sv}

    def tokens(i, codes, scale, h, a, n):
        """Positions a .. a + n of sequence i, one head."""
        pos = torch.arange(a, a + n, device=dev)
        page = s["page_table"][i][pos // size].long()
        c = codes[page, h, pos % size] if codes.dim() == 4 else codes[page, h, pos % size // 16, :, pos % 16]
        return c.double() * scale[page, h].double()[:, None]

    if case["op"] == "read":
        out = {x: torch.empty(s["tokens"], case["heads_kv"], case["dim"], dtype=torch.float64, device=dev) for x in "kv"}
        at = 0
        for i, (n, a) in enumerate(zip(new, full)):
            for h in range(case["heads_kv"]):
                for x in "kv":
                    out[x][at:at + n, h] = tokens(i, s[x], s[x + "_scale"], h, a, n)
            at += n
        return out
    heads, group = case["heads_kv"], case["heads_q"] // case["heads_kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    at = 0
    for i, (n, length) in enumerate(zip(new, full)):
        if n and length:
            key = torch.arange(length, device=dev)
            pos = torch.arange(length - n, length, device=dev)[:, None]
            hidden = key > pos
            if case["op"] == "sinks":
                hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
            for h in range(heads):
                k, v = (tokens(i, s[x], s[x + "_scale"], h, 0, length) for x in "kv")
                for j in range(h * group, (h + 1) * group):
                    w = (s["q"][at:at + n, j].double() @ k.T) / math.sqrt(case["dim"])
                    w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                    out[at:at + n, j] = torch.nan_to_num(w, nan=0.0) @ v  # a row that sees nothing is 0
        at += n
    return {"out": out}
