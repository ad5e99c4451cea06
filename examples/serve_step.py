"""One layer's attention as a serving loop runs it: prompts of mixed lengths are
rotated, appended to a paged 8-bit cache and attended to, then tokens are
generated one at a time, the step recorded in a HIP graph and replayed.

    python examples/serve_step.py [--steps 32]

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
PROMPTS = (700, 33, 1500, 1)


def reference(q, k, v, n):
    """softmax(q k / sqrt(dim)) v of the last n positions, causal, float64."""
    length = k.shape[0]
    k, v = (t.double().repeat_interleave(HEADS // KV_HEADS, 1).transpose(0, 1) for t in (k, v))
    s = q.double().transpose(0, 1) @ k.transpose(1, 2) / DIM ** 0.5
    seen = torch.arange(length, device=q.device) <= torch.arange(length - n, length, device=q.device)[:, None]
    return (torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ v).transpose(0, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=32)
    steps = ap.parse_args().steps
    pkg = __graft_entry__.load_package()
    dev = torch.device("cuda:0")
    torch.manual_seed(0)
    plan = pkg.plan_rotary(DIM, base=500000.0)
    batch = len(PROMPTS)
    width = max(-(-(n + steps) // PAGE) for n in PROMPTS)
    cache = pkg.PagedCache.empty(batch * width, KV_HEADS, DIM, PAGE, dev)
    table = torch.randperm(batch * width, device=dev).int().view(batch, width)

    def project(tokens):  # stands for a layer's fused projection
        return torch.randn(tokens, HEADS + 2 * KV_HEADS, DIM, device=dev, dtype=torch.bfloat16)

    def split(x):
        return x.split([HEADS, KV_HEADS, KV_HEADS], 1)

    # the prompts, all in one call
    offsets = torch.tensor([0, *torch.tensor(PROMPTS).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    starts = torch.zeros(batch, dtype=torch.int32, device=dev)
    lengths = torch.tensor(PROMPTS, dtype=torch.int32, device=dev)
    x = project(sum(PROMPTS))
    q, k, v = split(x)
    turned = pkg.append_paged_cache(cache, k, v, table, starts, offsets=offsets, rotary=plan, q=q)
    out = pkg.attend_paged_cache(cache, turned, table, lengths, offsets=offsets, max_length=max(PROMPTS))
    keys, values, worst, at = [], [], 0.0, 0
    for n in PROMPTS:
        rows = slice(at, at + n)
        keys.append(pkg.execute_rotary_plan(plan, k[rows], torch.arange(n, device=dev)))
        values.append(v[rows])
        want = reference(turned[rows], keys[-1], values[-1], n)
        worst = max(worst, float((out[rows].double() - want).norm() / want.norm()))
        at += n
    print(f"prompts of {PROMPTS} tokens: within {worst:.4f} of float64 on unrounded keys and values", flush=True)

    # generation: one step captured, then replayed
    after = lengths + 1
    x = project(batch)

    def step():
        q, k, v = split(x)
        turned = pkg.append_paged_cache(cache, k, v, table, lengths, rotary=plan, q=q)
        return turned, pkg.attend_paged_cache(cache, turned, table, after)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            turned, out = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    spent, worst = 0.0, 0.0
    for i in range(steps):
        x.copy_(project(batch))
        torch.cuda.synchronize()
        began = time.perf_counter()
        graph.replay()
        torch.cuda.synchronize()
        spent += time.perf_counter() - began
        _, k, v = split(x)
        for b in range(batch):
            keys[b] = torch.cat([keys[b], pkg.execute_rotary_plan(plan, k[b:b + 1], lengths[b:b + 1])])
            values[b] = torch.cat([values[b], v[b:b + 1]])
            want = reference(turned[b:b + 1], keys[b], values[b], 1)
            worst = max(worst, float((out[b:b + 1].double() - want).norm() / want.norm()))
        lengths += 1
        after += 1
    print(f"{steps} steps of {batch} sequences: within {worst:.4f}, {spent / max(1, steps) * 1e6:.1f} us a step, waited for")
    if not worst < 0.1:
        raise SystemExit("further off than an 8-bit cache explains")


if __name__ == "__main__":
    main()
