"""One layer's attention where conversations begin with the same picture: the
prompt's patches stand at (frame, row, column) positions, its pages are filled
once and shared by all conversations, whose own tokens follow; a step of all of
them is recorded in a HIP graph and replayed, once attending to everything and
once to a window and the first tokens; at the end a conversation is read back
out of the 8-bit cache.

    python examples/shared_prompt.py [--steps 16]

Prints how far each phase is from the same computed in float64 from unrounded
keys and values (what the 8-bit cache costs), and the time of a step.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import __graft_entry__  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE = 32, 8, 128, 64
GRID = (1, 24, 32)  # frames, rows and columns of the picture
SYSTEM = 40         # tokens of text before it
QUESTIONS = (90, 7, 200, 31, 1, 64)
WINDOW, SINKS = 256, 32


def reference(q, k, v, n, window=None, sinks=0):
    """softmax(q k / sqrt(dim)) v of the last n positions, causal, float64."""
    length = k.shape[0]
    k, v = (t.double().repeat_interleave(HEADS // KV_HEADS, 1).transpose(0, 1) for t in (k, v))
    s = q.double().transpose(0, 1) @ k.transpose(1, 2) / DIM ** 0.5
    key = torch.arange(length, device=q.device)
    own = torch.arange(length - n, length, device=q.device)[:, None]
    seen = key <= own
    if window:
        seen &= (key > own - window) | (key < sinks)
    return (torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v).transpose(0, 1)


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=16)
    steps = ap.parse_args().steps
    pkg = __graft_entry__.load_package()
    dev = torch.device("cuda:0")
    torch.manual_seed(0)
    # 64 pairs: 16 turned by the frame, 24 by the row, 24 by the column
    plan = pkg.plan_rotary(DIM, base=500000.0, axes=pkg.RotaryAxes((16, 24, 24)))
    batch = len(QUESTIONS)

    # Places: text counts up on all axes together, a picture's patches start
    # where the text before them ended, and the text after goes on from the
    # largest place used.
    frames, rows, columns = GRID
    grid = torch.stack(torch.meshgrid(*(torch.arange(n, device=dev) for n in GRID), indexing="ij")).reshape(3, -1)
    prompt_places = torch.cat([torch.arange(SYSTEM, device=dev).expand(3, -1), SYSTEM + grid], 1)
    prompt = prompt_places.shape[1]
    goes_on = int(prompt_places.max()) + 1
    shared = prompt // PAGE  # whole pages; the last tokens of a prompt are each conversation's own

    width = -(-(prompt + max(QUESTIONS) + steps) // PAGE)
    cache = pkg.PagedCache.empty(shared + batch * (width - shared), KV_HEADS, DIM, PAGE, dev)
    order = torch.randperm(cache.pages, device=dev).int()
    table = torch.cat([order[:shared].expand(batch, shared), order[shared:].view(batch, -1)], 1).contiguous()
    prefix_pages = torch.tensor([shared], dtype=torch.int32, device=dev)

    def project(tokens):  # stands for a layer's fused projection
        return torch.randn(tokens, HEADS + 2 * KV_HEADS, DIM, device=dev, dtype=torch.bfloat16)

    def split(x):
        return x.split([HEADS, KV_HEADS, KV_HEADS], 1)

    def int32(*values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    # the whole pages of the prompt, once, through the first conversation's row of the table
    px = project(prompt)
    pq, pk, pv = split(px)
    whole = shared * PAGE
    turned = pkg.append_paged_cache(cache, pk[:whole], pv[:whole], table[:1], int32(0), offsets=int32(0, whole), rotary=plan, q=pq[:whole],
                                    positions=prompt_places[:, :whole])
    out = pkg.attend_paged_cache(cache, turned, table[:1], int32(whole))
    prompt_keys = pkg.execute_rotary_plan(plan, pk, prompt_places)
    worst = off(out, reference(turned, prompt_keys[:whole], pv[:whole], whole))
    print(f"a prompt of {SYSTEM} tokens and {frames} x {rows} x {columns} patches: within {worst:.4f} of float64", flush=True)

    # the rest of it and the questions, all conversations in one call
    tail = prompt - whole
    counts = [tail + n for n in QUESTIONS]
    offsets = int32(0, *torch.tensor(counts).cumsum(0).tolist())
    x = torch.cat([torch.cat([px[whole:], project(n)]) for n in QUESTIONS])
    places = torch.cat([torch.cat([prompt_places[:, whole:], goes_on + torch.arange(n, device=dev).expand(3, -1)], 1) for n in QUESTIONS], 1)
    q, k, v = split(x)
    turned = pkg.append_paged_cache(cache, k, v, table, int32(*[whole] * batch), offsets=offsets, rotary=plan, q=q, positions=places)
    lengths = int32(*[whole + n for n in counts])
    out = pkg.attend_paged_cache(cache, turned, table, lengths, offsets=offsets, max_length=whole + max(counts), prefix_pages=prefix_pages)
    own = pkg.execute_rotary_plan(plan, k, places)
    keys, values, at = [], [], 0
    for n in counts:
        part = slice(at, at + n)
        keys.append(torch.cat([prompt_keys[:whole], own[part]]))
        values.append(torch.cat([pv[:whole], v[part]]))
        worst = max(worst, off(out[part], reference(turned[part], keys[-1], values[-1], n)))
        at += n
    print(f"questions of {QUESTIONS} tokens behind it: within {worst:.4f}", flush=True)

    # generation: one step captured, then replayed
    after = lengths + 1
    place = goes_on + int32(*QUESTIONS).expand(3, -1).contiguous()
    x = project(batch)

    def step():
        q, k, v = split(x)
        turned = pkg.append_paged_cache(cache, k, v, table, lengths, rotary=plan, q=q, positions=place)
        return (turned, pkg.attend_paged_cache(cache, turned, table, after, prefix_pages=prefix_pages),
                pkg.attend_paged_cache(cache, turned, table, after, window=WINDOW, sinks=SINKS))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            turned, all_seen, windowed = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    spent = 0.0
    for _ in range(steps):
        x.copy_(project(batch))
        torch.cuda.synchronize()
        began = time.perf_counter()
        graph.replay()
        torch.cuda.synchronize()
        spent += time.perf_counter() - began
        _, k, v = split(x)
        new = pkg.execute_rotary_plan(plan, k, place)
        for b in range(batch):
            row = slice(b, b + 1)
            keys[b] = torch.cat([keys[b], new[row]])
            values[b] = torch.cat([values[b], v[row]])
            worst = max(worst, off(all_seen[row], reference(turned[row], keys[b], values[b], 1)),
                        off(windowed[row], reference(turned[row], keys[b], values[b], 1, WINDOW, SINKS)))
        lengths += 1
        after += 1
        place += 1
    print(f"{steps} steps of {batch} conversations: within {worst:.4f}, {spent / max(1, steps) * 1e6:.1f} us a step, waited for", flush=True)

    # a conversation's own tokens out of the cache, to be moved or trained on
    count = int(lengths[0]) - whole
    k, v = pkg.read_paged_cache(cache, table[:1], int32(whole), count, offsets=int32(0, count))
    back = max(off(k, keys[0][whole:].double()), off(v, values[0][whole:].double()))
    print(f"{count} tokens read back: within {back:.4f}")
    if not max(worst, back) < 0.1:
        raise SystemExit("further off than an 8-bit cache explains")


if __name__ == "__main__":
    main()
