"""A serving step through the paged cache, operator by operator.

For each kind of step (single tokens of one request or of a batch, a chunk of a
long prompt, both at once, with and without a window) this fills a ``PagedCache``
with requests of the given lengths and prints the device time (HIP events around
``--steps`` calls after ``--warmup``) of the step's page plan, of storing its keys
and values with q and k rotated, and of the attention, with the attention's
rates: bytes of visible K and V, q and o, and 4 * 128 FLOP for each (row, visible
key) pair of a head.

Usage: python -m fa_amd.measure.serving [--dtype float16|bfloat16] [--page-size N] [--steps N]
"""

from __future__ import annotations

import argparse
from dataclasses import dataclass


@dataclass(frozen=True)
class Step:
    name: str
    heads_q: int
    heads_kv: int
    spans: tuple            # (earlier tokens, new tokens) of every request
    window: "int | None" = None
    sinks: int = 0


STEPS = (
    Step("one request", 12, 1, ((4098, 1),)),
    Step("one long request", 12, 1, ((131071, 1),)),
    Step("64 requests", 64, 8, tuple((125 * (i + 1), 1) for i in range(64))),
    Step("chunk of a prompt", 12, 1, ((30001, 2048),)),
    Step("two chunks, 22 tokens", 32, 8, ((5000, 1000), (9000, 1000)) + ((4000, 1),) * 22, 4096, 4),
)


def visible_pairs(past, new, window, sinks):
    """(row, key) pairs that rows at positions past .. past + new - 1 see."""
    total = 0
    for p in range(past, past + new):
        total += p + 1 if window is None else min(p + 1, window + min(sinks, max(0, p + 1 - window)))
    return total


def work(step):
    """(bytes, FLOP) that the step's attention cannot do without."""
    keys = pairs = 0
    for past, new in step.spans:
        first = 0 if step.window is None else max(0, past - step.window + 1)
        keys += past + new - first + min(step.sinks, first)
        pairs += visible_pairs(past, new, step.window, step.sinks)
    rows = sum(new for _, new in step.spans) * step.heads_q
    return 512 * (rows + keys * step.heads_kv), 512 * step.heads_q * pairs


def measure(step, dtype, page_size, warmup, steps):
    import torch

    from fa_amd.cache import CacheConfig, PagedCache
    from fa_amd.harness import timing
    from fa_amd.serving import PagedConfig

    longest = max(p + n for p, n in step.spans)
    pages = sum(-(-(p + n) // page_size) for p, n in step.spans)
    cache = PagedCache(CacheConfig(
        layers=1, heads_q=step.heads_q, heads_kv=step.heads_kv, pages=pages, page_size=page_size,
        max_batch=len(step.spans), max_length=longest, dtype=dtype,
        attention=PagedConfig(window=step.window, sinks=step.sinks)))
    cache.k.normal_()
    cache.v.normal_()
    # The requests' earlier tokens: pages and lengths, random keys and values.
    past = torch.tensor([p for p, _ in step.spans], dtype=torch.int32, device="cuda")
    new = torch.tensor([n for _, n in step.spans], dtype=torch.int32, device="cuda")
    cache.begin(past, 0, 1)
    tokens, max_new = sum(n for _, n in step.spans), max(n for _, n in step.spans)
    q, k, v = (torch.randn(tokens, h, 128, device="cuda").to(getattr(torch, dtype))
               for h in (step.heads_q, step.heads_kv, step.heads_kv))
    lengths, taken = cache.lengths.clone(), cache.taken.clone()
    plan = cache.begin(new, tokens, max_new)

    def us(call):
        return timing.device_us(call, iters=steps, warmup=warmup)

    moved, flops = work(step)
    attend = us(lambda: cache.attention(q, cache.k[0], cache.v[0], cache.table, plan.query_starts,
                                        plan.key_lengths, max_new))
    return {
        "name": step.name,
        "plan": us(lambda: cache.planner(lengths, new, cache.table, cache.pages[:-1], taken, tokens)),
        "store": us(lambda: cache.rotary.append(q, k, v, plan.positions, plan.slots, cache.k[0],
                                                cache.v[0])),
        "attend": attend,
        "tbs": moved / attend / 1e6,
        "tflops": flops / attend / 1e6,
    }


def render(rows, dtype, command):
    lines = [f"serving step, {dtype}: us an operator call", f"command: {command}",
             f"{'step':24s} {'plan':>8s} {'store':>8s} {'attend':>9s} {'TB/s':>6s} {'TFLOP/s':>8s}"]
    for r in rows:
        lines.append(f"{r['name']:24s} {r['plan']:8.1f} {r['store']:8.1f} {r['attend']:9.1f} "
                     f"{r['tbs']:6.2f} {r['tflops']:8.1f}")
    return lines


def main(argv=None):
    ap = argparse.ArgumentParser(prog="python -m fa_amd.measure.serving",
                                 description=__doc__.splitlines()[0])
    ap.add_argument("--dtype", default="float16", choices=("float16", "bfloat16"))
    ap.add_argument("--page-size", type=int, default=64)
    ap.add_argument("--warmup", type=int, default=10)
    ap.add_argument("--steps", type=int, default=50)
    args = ap.parse_args(argv)
    rows = [measure(s, args.dtype, args.page_size, args.warmup, args.steps) for s in STEPS]
    command = f"python -m fa_amd.measure.serving --dtype {args.dtype} --page-size {args.page_size}"
    print("\n".join(render(rows, args.dtype, command)))


if __name__ == "__main__":
    main()
