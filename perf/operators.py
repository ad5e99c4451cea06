"""The language-model operators whose time is measured, as a user's program runs them.

* ``rotary``: positions rotated into query and key heads (``plan_rotary``,
  ``execute_rotary_plan``), with the gradient where the case trains;
* ``append``: new keys and values written to a paged 8-bit cache, the keys
  (and the step's queries) rotated on the way (``append_paged_cache``);
* ``attend``: attention over that cache (``attend_paged_cache``).

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
heads; head dims 64, 96, 128 and 256; pages of 16 to 128 tokens.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

MAX_POSITIONS = 1 << 20
BASE = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ----------------------------------------------------------------

def _rotary(batch, seq, heads, dim, rot, layout, dtype, scaling="none", train=False, extra=0, first=0) -> dict:
    """``extra`` heads lie between one token's heads and the next one's (the
    input is a view of a larger projection); positions start at ``first``."""
    return {"op": "rotary", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
            "dtype": dtype, "scaling": scaling, "train": train, "extra": extra, "first": first}


def _append(seqs, new, cached, heads_q, heads_kv, dim, page, dtype, layout="half", rot=None) -> dict:
    """``new`` tokens a sequence (1: each exactly one; more: the mean of mixed
    counts) onto up to ``cached`` tokens each."""
    return {"op": "append", "seqs": seqs, "new": new, "cached": cached, "heads_q": heads_q, "heads_kv": heads_kv,
            "dim": dim, "page": page, "dtype": dtype, "layout": layout, "rot": dim if rot is None else rot}


def _attend(seqs, new, context, heads_q, heads_kv, dim, page, dtype, window=0, mixed=False) -> dict:
    """``new`` queries a sequence, the last positions of contexts of up to
    ``context`` tokens (``mixed``: of any length up to it, some empty)."""
    return {"op": "attend", "seqs": seqs, "new": new, "context": context, "heads_q": heads_q, "heads_kv": heads_kv,
            "dim": dim, "page": page, "dtype": dtype, "window": window, "mixed": mixed}


def listed() -> list:
    return [
        # the query and key heads of one token, a view of its fused projection: one step of an interactive reply
        {"name": "rotary_token", **_rotary(1, 1, 40, 128, 128, "half", "bf16", extra=8, first=1000)},
        # a training batch, forward and gradient
        {"name": "rotary_train", **_rotary(2, 4096, 32, 128, 128, "half", "bf16", train=True)},
        # one very long document whose positions were scaled, half of each head rotated, in 32 bits, odd length
        {"name": "rotary_long_parts", **_rotary(1, 100003, 8, 96, 48, "interleaved", "fp32", "parts", True, 0, 900000)},
        # one token into one sequence's cache: the smallest step of serving
        {"name": "append_token", **_append(1, 1, 777, 32, 8, 128, 64, "bf16")},
        # a full serving batch, one token each
        {"name": "append_batch", **_append(256, 1, 8192, 32, 8, 128, 64, "bf16")},
        # several prompts of mixed odd lengths, part of each head rotated, short pages
        {"name": "append_mixed", **_append(13, 700, 500, 28, 4, 64, 16, "fp16", "interleaved", 32)},
        # four long prompts at once: bandwidth
        {"name": "append_bulk", **_append(4, 8192, 0, 32, 8, 128, 64, "bf16")},
        # one token's attention over a short reply: latency
        {"name": "attend_token", **_attend(1, 1, 1000, 32, 8, 128, 64, "bf16")},
        # a serving batch of mixed lengths, empty slots among them, seven query heads a key head
        {"name": "attend_mixed", **_attend(64, 1, 8192, 28, 4, 128, 16, "fp16", mixed=True)},
        # one token over a very long context: the cache is read once, by the whole chip
        {"name": "attend_long", **_attend(1, 1, 1 << 18, 32, 8, 128, 64, "bf16")},
        # several drafted tokens a sequence checked at once, within a window
        {"name": "attend_verify", **_attend(32, 5, 4096, 64, 8, 64, 32, "bf16", window=1500)},
        # a piece of a long prompt against what is cached: matrix products
        {"name": "attend_chunk", **_attend(1, 2048, 32768, 32, 8, 128, 64, "bf16")},
    ]


def _log(rng, low, high) -> int:
    return max(low, min(high, int(2.0 ** rng.uniform(math.log2(low), math.log2(high + 1)))))


def draw(rng) -> dict:
    op = rng.choice(["rotary", "append", "attend", "attend"])
    dim = rng.choice([64, 96, 128, 128, 256])
    if op == "rotary":
        batch = _log(rng, 1, 64)
        heads = rng.randint(1, 64)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        # at most 2^28 values
        seq = _log(rng, 1, max(1, min(131072, (1 << 28) // (batch * heads * dim))))
        rot = rng.choice([dim, dim, dim // 2, dim // 4, 20])
        return _rotary(batch, seq, heads, dim, rot, rng.choice(["half", "interleaved"]), dtype,
                       rng.choice(["none", "linear", "parts"]), rng.random() < 0.5, rng.choice([0, 0, 8]),
                       rng.choice([0, 0, _log(rng, 1, MAX_POSITIONS - 131072)]))
    heads_kv = rng.choice([1, 2, 4, 8, 16])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 7, 8] if heads_kv <= 8 else [1, 2, 4])
    page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "fp16"])
    seqs = _log(rng, 1, 256)
    if op == "append":
        # at most 2^27 values of q
        most = max(1, min(8192, (1 << 27) // (seqs * heads_q * dim)))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, most)
        return _append(seqs, new, _log(rng, 1, 8192), heads_q, heads_kv, dim, page,
                       rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["half", "interleaved"]),
                       rng.choice([dim, dim, dim // 2, 20]))
    new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 2048)])
    # at most 2^29 bytes of cache and 2^39 operations a product
    most = min(1 << 18, (1 << 28) // (seqs * heads_kv * dim), (1 << 38) // (seqs * new * heads_q * dim))
    context = _log(rng, 1, max(1, most))
    new = min(new, context)
    return _attend(seqs, new, context, heads_q, heads_kv, dim, page, dtype,
                   rng.choice([0, 0, 0, _log(rng, 1, 4096)]), rng.random() < 0.5)


# ---- sizes a case fixes ---------------------------------------------------

def _lengths(case):
    """(new tokens, cached tokens before them) of each sequence; they follow
    from the case alone, so that every seed's inputs are the same work."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["seqs"]
    if case["op"] == "append":
        new = [1 if case["new"] == 1 else r.randint(1, 2 * case["new"] - 1) for _ in range(n)]
        if case["cached"] == 0:
            new = [case["new"]] * n
        return new, [r.randint(0, case["cached"]) for _ in range(n)]
    new = [case["new"]] * n
    full = [case["context"]] * n
    if case["mixed"]:
        full = [r.choice([0, case["context"]]) if r.random() < 0.1 else r.randint(1, case["context"]) for _ in range(n)]
        if case["new"] > 1:
            new = [r.randint(0, case["new"]) for _ in range(n)]
        full[0], new[0] = case["context"], case["new"]
    return new, full


def _frequencies(case):
    """(radians a position of each pair, amplitude), in 64 bits."""
    r = case["rot"]
    theta = [BASE ** (-2.0 * j / r) for j in range(r // 2)]
    kind = case.get("scaling", "none")
    if kind == "linear":
        return [t / 4.0 for t in theta], 1.0
    if kind == "parts":
        out = []
        for t in theta:
            g = min(1.0, max(0.0, (8192 * t / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
            out.append(t * (g + (1.0 - g) / 16.0))
        return out, 0.1 * math.log(16.0) + 1.0
    return theta, 1.0


@functools.lru_cache(maxsize=4)
def _table(freqs, amplitude, positions, device):
    """cos and sin of every position, made in 64 bits: what a program without
    this library keeps beside the model."""
    a = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * torch.tensor(
        freqs, device=device, dtype=torch.float64)
    return (a.cos() * amplitude).float(), (a.sin() * amplitude).float()


# ---- inputs ---------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device())


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
    pages anywhere in the pool, unused entries -1."""
    dev, size = _device(), case["page"]
    need = [-(-n // size) for n in full]
    pool = sum(need) + 3
    k, ks = _random_pages(g, pool, case["heads_kv"], (size, case["dim"]))
    v, vs = _random_pages(g, pool, case["heads_kv"], (size // 16, case["dim"], 16))
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    width = max(1, max(need))
    count = torch.tensor(need, device=dev)
    at = torch.arange(width, device=dev)
    first = torch.cumsum(count, 0) - count
    table = order[(first[:, None] + at[None]).clamp(max=pool - 1)]
    table = torch.where(at[None] < count[:, None], table, torch.full_like(table, -1))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "page_table": table.contiguous()}


def _offsets(new):
    c = [0]
    for n in new:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=_device())


def prepare(case: dict, seed: int) -> dict:
    dev = _device()
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev).to(dt)

    s = {"case": case}
    if op == "rotary":
        b, n, h, d = case["batch"], case["seq"], case["heads"], case["dim"]
        s["x"] = randn(b, n, h + case["extra"], d)[:, :, :h]
        most = min(MAX_POSITIONS - n, case["first"] + 1000)
        first = torch.randint(min(case["first"], most), most + 1, (b, 1), generator=g, device=dev)
        s["positions"] = first + torch.arange(n, device=dev)
        if case["train"]:
            s["x"].requires_grad_()
            s["grad"] = randn(b, n, h, d)
        s["roots"] = _table(*map(_frozen, _frequencies(case)), MAX_POSITIONS, dev)
        return s
    new, full = _lengths(case)
    t = sum(new)
    if op == "append":
        s |= _paged(g, case, [a + b for a, b in zip(new, full)])
        fused = randn(t, case["heads_q"] + 2 * case["heads_kv"], case["dim"])  # one projection's output
        s["q"], s["new_k"], s["new_v"] = fused.split([case["heads_q"], case["heads_kv"], case["heads_kv"]], dim=1)
        s["starts"] = torch.tensor(full, dtype=torch.int32, device=dev)
        s["roots"] = _table(*map(_frozen, _frequencies(case)), MAX_POSITIONS, dev)
    else:
        s |= _paged(g, case, full)
        s["q"] = randn(t, case["heads_q"], case["dim"])
        s["lengths"] = torch.tensor(full, dtype=torch.int32, device=dev)
        s["max_length"], s["max_new"] = max(full), max(new)
    s["offsets"] = None if all(n == 1 for n in new) else _offsets(new)
    return s


def _frozen(v):
    return tuple(v) if isinstance(v, list) else v


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


def _plain_rotary(s):
    c, x = s["case"], s["x"].detach()
    cos, sin = (t[s["positions"]][:, :, None] for t in s["roots"])
    y = _rotated(x, cos, sin, c["layout"]).to(x.dtype)
    if not c["train"]:
        return {"y": y}
    return {"y": y, "x_grad": _rotated(s["grad"], cos, -sin, c["layout"]).to(x.dtype)}


def _sequence_of(offsets, tokens, sequences):
    """Which sequence each token belongs to, and its place in it."""
    dev = _device()
    if offsets is None:
        return torch.arange(sequences, device=dev), torch.zeros(sequences, dtype=torch.int64, device=dev)
    at = torch.arange(tokens, device=dev)
    seq = torch.searchsorted(offsets[1:], at, right=True)
    return seq, at - offsets[seq]


def _plain_append(s):
    c, k, v = s["case"], s["new_k"], s["new_v"]
    size, t = c["page"], k.shape[0]
    starts = s["starts"].long()
    seq, place = _sequence_of(s["offsets"], t, starts.numel())
    pos = starts[seq] + place
    cos, sin = (r[pos][:, None] for r in s["roots"])
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


def _plain_attend(s):
    c, q = s["case"], s["q"]
    size, dim, hk = c["page"], c["dim"], c["heads_kv"]
    group, n = c["heads_q"] // hk, s["max_new"]
    b, t = s["page_table"].shape[0], q.shape[0]
    pages = s["page_table"].clamp(min=0).long()
    length = pages.shape[1] * size
    k = s["k"][pages].float() * s["k_scale"][pages][..., None, None]
    k = k.transpose(1, 2).reshape(b, hk, length, dim)
    v = s["v"][pages].float() * s["v_scale"][pages][..., None, None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(b, hk, length, dim)
    seq, place = _sequence_of(s["offsets"], t, b)
    count = torch.ones(b, dtype=torch.int64, device=q.device) if s["offsets"] is None else s["offsets"].diff().long()
    padded = torch.zeros(b, n, hk, group, dim, device=q.device)
    padded[seq, place] = q.float().reshape(t, hk, group, dim)
    rows = padded.permute(0, 2, 1, 3, 4).reshape(b, hk, n * group, dim)
    score = torch.matmul(rows, k.transpose(-1, -2).contiguous()) * dim ** -0.5
    at = torch.arange(length, device=q.device)
    pos = (s["lengths"] - count)[:, None] + torch.arange(n, device=q.device)  # [b][n]
    seen = at <= pos[..., None]
    if c["window"]:
        seen &= at > pos[..., None] - c["window"]
    seen = seen[:, None, :, None].expand(b, 1, n, group, length).reshape(b, 1, n * group, length)
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    # what lies past a sequence's end is not its own
    out = torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)
    out = out.reshape(b, hk, n, group, dim).permute(0, 2, 1, 3, 4)
    return {"out": out[seq, place].reshape(t, c["heads_q"], dim).to(q.dtype)}


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _rotary_plan(pkg, case):
    kind = case.get("scaling", "none")
    scaling = {"none": None, "linear": ("linear", 4.0),
               "parts": ("parts", 16.0, 8192, 1.0, 32.0, 0.1 * math.log(16.0) + 1.0)}[kind]
    return pkg.plan_rotary(case["dim"], rot_dim=case["rot"], layout=case["layout"], base=BASE,
                           scaling=None if scaling is None else pkg.RotaryScaling(*scaling),
                           max_positions=MAX_POSITIONS)


def _own_pass(s):
    pkg, c = _package(), s["case"]
    if "plan" not in s:  # the handles a program keeps beside its tensors
        s["plan"] = _rotary_plan(pkg, c) if c["op"] != "attend" else None
        s["cache"] = pkg.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"]) if c["op"] != "rotary" else None
    if c["op"] == "rotary":
        y = pkg.execute_rotary_plan(s["plan"], s["x"], s["positions"])
        if not c["train"]:
            return {"y": y}
        return {"y": y.detach(), "x_grad": torch.autograd.grad(y, s["x"], s["grad"])[0]}
    if c["op"] == "append":
        q = pkg.append_paged_cache(s["cache"], s["new_k"], s["new_v"], s["page_table"], s["starts"],
                                   offsets=s["offsets"], rotary=s["plan"], q=s["q"])
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"out": pkg.attend_paged_cache(s["cache"], s["q"], s["page_table"], s["lengths"], offsets=s["offsets"],
                                          max_length=s["max_length"],
                                          window=c["window"] or None)}


def run(state: dict):
    if own:
        return _own_pass(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[state["case"]["op"]](state)


def _seen(case):
    """(keys that any query of a sequence sees, query and key pairs) over all sequences."""
    keys = pairs = 0
    w = case["window"]
    for n, length in zip(*_lengths(case)):
        first = max(0, length - n)  # position of the first query that sees anything
        top = length
        if top <= first or not n:
            continue
        low = max(0, first - w + 1) if w else 0
        keys += top - low
        full = top * (top + 1) // 2 - first * (first + 1) // 2
        if w:  # of position p: min(p + 1, w)
            cut = max(first, w)
            if cut < top:
                full -= (top - w) * (top - w + 1) // 2 - (cut - w) * (cut - w + 1) // 2
        pairs += full
    return keys, pairs


def work(case: dict) -> dict:
    """Each input read once, each output written once: the rotated heads and
    their gradient (6 operations a pair); the new keys, values and queries and
    their codes; the visible codes with their scales, the queries and outputs
    (two products of ``dim`` for a query head and key that see each other)."""
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "rotary":
        tokens = case["batch"] * case["seq"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * tokens * (2 * case["heads"] * case["dim"] * size + 8),
                "flops": passes * tokens * case["heads"] * 3 * case["rot"]}
    if case["op"] == "append":
        t = sum(_lengths(case)[0])
        kv = 2 * case["heads_kv"] * case["dim"]
        return {"bytes": t * (kv * (size + 1) + 2 * case["heads_q"] * case["dim"] * size),
                "flops": t * (3 * (case["heads_q"] + case["heads_kv"]) * case["rot"] + 2 * kv)}
    keys, pairs = _seen(case)
    t = sum(_lengths(case)[0])
    return {"bytes": keys * case["heads_kv"] * (2 * case["dim"] + 8.0 / case["page"])
            + 2 * t * case["heads_q"] * case["dim"] * size,
            "flops": 4 * pairs * case["heads_q"] * case["dim"]}


# ---- in 64 bits -----------------------------------------------------------

def _turn64(x, pos, case):
    """x [tokens, heads, dim] as complex pairs times m exp(i pos theta)."""
    freqs, m = _frequencies(case)
    p = len(freqs)
    a = pos.double()[:, None] * torch.tensor(freqs, device=x.device, dtype=torch.float64)
    root = torch.polar(torch.full_like(a, m), a)[:, None]
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
        pos = s["positions"].reshape(-1)
        out = {"y": _turn64(s["x"].detach().reshape(-1, h, d), pos, case).reshape(b, n, h, d)}
        if case["train"]:
            out["x_grad"] = _turn64(s["grad"].reshape(-1, h, d), -pos, case).reshape(b, n, h, d)
        return out
    new, full = _lengths(case)
    size = case["page"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(a, a + n, device=_device()) for n, a in zip(new, full)])
        k, v = _turn64(s["new_k"], pos, case), s["new_v"].double()
        ck, cv = s["k"].double(), s["v"].double()
        sk, sv = s["k_scale"].double(), s["v_scale"].double()
        at = 0
        for i, (n, a) in enumerate(zip(new, full)):
            p = a
            while p < a + n:  # one page at a time
                m = min(size - p % size, a + n - p)
                page, o = int(s["page_table"][i, p // size]), p % size
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
        return {"q": _turn64(s["q"], pos, case), "k": ck, "v": cv, "k_scale": sk, "v_scale": sv}
    heads, group = case["heads_kv"], case["heads_q"] // case["heads_kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for i, (n, length) in enumerate(zip(new, full)):
        if n and length:
            pages = s["page_table"][i, :-(-length // size)].long()
            key = torch.arange(length, device=out.device)
            pos = torch.arange(length - n, length, device=out.device)[:, None]
            hidden = key > pos
            if case["window"]:
                hidden |= key <= pos - case["window"]
            for h in range(heads):
                k = (s["k"][pages, h].double() * s["k_scale"][pages, h, None, None].double()).reshape(-1, case["dim"])
                v = s["v"][pages, h].double() * s["v_scale"][pages, h, None, None, None].double()
                v = v.transpose(-1, -2).reshape(-1, case["dim"])[:length]
                for j in range(h * group, (h + 1) * group):
                    w = (s["q"][at:at + n, j].double() @ k[:length].T) / math.sqrt(case["dim"])
                    w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                    out[at:at + n, j] = torch.nan_to_num(w, nan=0.0) @ v  # a row that sees nothing is 0
        at += n
    return {"out": out}
