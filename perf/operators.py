"""Performance cases of the serving operators: block tables and slot maps built
from request lengths, rotary positions written into a paged cache, attention
over that cache, and attention with a sliding window and sinks.

A case has an ``op`` and the sizes of one call:

  plan     ``batch`` requests take pages of ``page`` tokens for their new ones
  rotary   ``tokens`` rows of q, k and v: q rotated, k rotated and stored with
           v in the pages that the slots name
  paged    attention of every request's new tokens over its pages
  window   attention with a window on contiguous [B, H, N, 128] tensors

The lengths of a ragged batch follow from the case's numbers alone (see
``_lengths``), what the tensors hold from the seed.
"""

import math
import random

import torch

own = False

DIM = 128
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _plan(batch, past_lo, past_hi, new, chunks, page, slack=0):
    return {"op": "plan", "batch": batch, "past_lo": past_lo, "past_hi": past_hi, "new": new,
            "chunks": chunks, "page": page, "slack": slack}


def _rotary(tokens, heads_q, heads_kv, page, dtype, layout, rotary, far, scaled):
    return {"op": "rotary", "tokens": tokens, "heads_q": heads_q, "heads_kv": heads_kv,
            "page": page, "dtype": dtype, "layout": layout, "rotary": rotary, "far": far,
            "scaled": scaled}


def _paged(batch, heads_q, heads_kv, past_lo, past_hi, new, chunks, page, dtype, window=0, sinks=0,
           lse=False):
    return {"op": "paged", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv,
            "past_lo": past_lo, "past_hi": past_hi, "new": new, "chunks": chunks, "page": page,
            "dtype": dtype, "window": window, "sinks": sinks, "lse": lse}


def _window(batch, heads_q, heads_kv, seq_q, seq_k, window, sinks, dtype, layout="bhnd", lse=False):
    return {"op": "window", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv,
            "seq_q": seq_q, "seq_k": seq_k, "window": window, "sinks": sinks, "dtype": dtype,
            "layout": layout, "lse": lse}


def listed():
    cases = {
        # The start of a decode step of a serving batch: one token a request.
        "plan_decode": _plan(48, 1, 8192, 1, 0, 16),
        # The start of a step that takes in many prompts beside decoding
        # requests, its token buffers padded to a fixed length.
        "plan_prompts": _plan(300, 1, 4096, 700, 90, 64, slack=555),
        # A decode step's rows: 48 single tokens, one KV head, whole heads
        # rotated in halves.
        "rotary_decode": _rotary(48, 12, 1, 16, "fp16", "half", 128, 131072, False),
        # A long prompt's rows: interleaved pairs in half of every head,
        # positions scaled for a longer context than the model was made for.
        "rotary_prompt": _rotary(40007, 32, 8, 64, "bf16", "interleaved", 64, 131072, True),
        # One request early in a generation, pages of 16: the smallest call.
        "paged_decode_4k": _paged(1, 12, 1, 4098, 4098, 1, 0, 16, "fp16"),
        # One request behind the longest context.
        "paged_decode_131k": _paged(1, 12, 1, 131071, 131071, 1, 0, 64, "fp16"),
        # A decode step of a serving batch, every context of another length.
        "paged_batch": _paged(64, 64, 8, 100, 8005, 1, 0, 32, "bf16"),
        # One chunk of a long prompt that is taken in pieces.
        "paged_chunk": _paged(1, 12, 1, 30001, 30001, 2048, 1, 64, "fp16", lse=True),
        # Decoding requests and two prompt chunks in one step, attention
        # limited to a window and the first tokens.
        "paged_mixed": _paged(24, 32, 8, 600, 12000, 1000, 2, 16, "bf16", window=4096, sinks=4),
        # One token each for eight requests, a window of a contiguous cache.
        "window_decode": _window(8, 64, 8, 1, 8005, 1024, 16, "fp16"),
        # A batch of prompts in the sequence-major layout, with the
        # log-sum-exp a merge needs.
        "window_batch": _window(4, 32, 8, 2048, 2048, 512, 0, "bf16", layout="bnhd", lse=True),
        # A 32768-token prompt, a window of 4096 and four sinks.
        "window_prompt": _window(1, 12, 1, 32768, 32768, 4096, 4, "fp16"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


HEADS = [(12, 1), (12, 1), (8, 1), (24, 2), (32, 8), (64, 8), (16, 16)]
MAX_BYTES = 1.0e9          # K and V of a drawn case
MAX_FLOPS = 3.0e11


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], both ends included."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "paged", "paged", "paged", "window", "window"])
    dtype = rng.choice(["fp16", "bf16"])
    heads_q, heads_kv = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "plan":
        batch = _log(rng, 1, 300)
        chunks = rng.choice([0, rng.randint(0, batch)])
        return _plan(batch, 1, _log(rng, 2, 8192), _log(rng, 1, 60000 // max(chunks, 90)), chunks,
                     page, slack=rng.choice([0, rng.randint(1, 600)]))
    if op == "rotary":
        tokens = min(_log(rng, 1, 120000), 40007 * 48 // (heads_q + 2 * heads_kv))
        return _rotary(tokens, heads_q, heads_kv, page, dtype, rng.choice(["half", "interleaved"]),
                       rng.choice([32, 64, 96, 128]), 131072, rng.random() < 0.4)
    while True:
        if op == "paged":
            batch = _log(rng, 1, 64)
            chunks = rng.choice([0, 0, min(batch, rng.randint(1, 3))])
            hi = _log(rng, 16, 131071)
            window = rng.choice([0, 0, _log(rng, 64, 8192)])
            case = _paged(batch, heads_q, heads_kv, max(1, hi // rng.choice([1, 4, 64])), hi,
                          _log(rng, 2, 2048), chunks, page, dtype, window=window,
                          sinks=_log(rng, 1, 64) if window and rng.random() < 0.5 else 0,
                          lse=rng.random() < 0.3)
            stored = sum(map(sum, _lengths(case)))
        else:
            decode = rng.random() < 0.4
            seq_k = _log(rng, 64, 65536)
            seq_q = rng.randint(1, 4) if decode else seq_k - (rng.randint(0, seq_k // 2)
                                                              if rng.random() < 0.3 else 0)
            batch = _log(rng, 1, 16)
            case = _window(batch, heads_q, heads_kv, seq_q, seq_k, _log(rng, 32, 8192),
                           rng.choice([0, _log(rng, 1, 64)]), dtype,
                           layout=rng.choice(["bhnd", "bnhd"]), lse=rng.random() < 0.3)
            stored = batch * (seq_k + seq_q * heads_q // heads_kv)
        if stored * heads_kv * DIM * 4 <= MAX_BYTES and work(case)["flops"] <= MAX_FLOPS:
            return case


def _lengths(case):
    """Tokens already stored and new tokens of every request: earlier lengths
    spread over the logarithm of their range, the first ``chunks`` requests
    with about ``new`` new tokens and the others with one."""
    rng = random.Random(case["batch"] * 1000003 + case["past_hi"] * 101 + case["new"])
    past = [_log(rng, case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]
    new = [max(1, case["new"] - rng.randint(0, case["new"] // 4)) if case["batch"] > 1 and
           i < case["chunks"] else case["new"] if i < case["chunks"] else 1
           for i in range(case["batch"])]
    return past, new


def _pages(case, length):
    return -(-length // case["page"])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(case):
    """Rotation per position of every pair, in 64 bits, and the factor on the
    rotated values. Scaled: positions compressed by 8 where a pair turns fewer
    than once over the 4096 positions of the original context, left alone
    where it turns more than 32 times, in between in proportion."""
    half = case["rotary"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    if not case["scaled"]:
        return freq, 1.0
    turns = torch.arange(half, dtype=torch.float64)
    lo = half * math.log(4096 / (32 * 2 * math.pi)) / math.log(10000.0)
    hi = half * math.log(4096 / (1 * 2 * math.pi)) / math.log(10000.0)
    ramp = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
    return freq / 8.0 * ramp + freq * (1.0 - ramp), 0.1 * math.log(8.0) + 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(
            TYPES[case["dtype"]])

    def shuffled(n):
        return torch.randperm(n, generator=gen, device="cuda").to(torch.int32)

    state = {"case": case}
    if case["op"] == "plan":
        past, new = _lengths(case)
        # Other seeds: the same requests in another order.
        order = torch.randperm(case["batch"], generator=gen, device="cuda").tolist()
        past, new = [past[i] for i in order], [new[i] for i in order]
        held = [_pages(case, n) for n in past]
        total = sum(_pages(case, p + n) for p, n in zip(past, new))
        pool = shuffled(total + 64)
        width = max(_pages(case, p + n) for p, n in zip(past, new)) + 3
        table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(held):
            table[b, :n] = pool[at:at + n]
            at += n
        state.update(past=_ints(past), new=_ints(new), table=table, pages=pool[at:].contiguous(),
                     taken=_ints([5]), tokens=sum(new) + case["slack"])
        if own:
            from fa_amd.serving import PagePlanner
            state["own"] = PagePlanner(page_size=case["page"])
        return state
    if case["op"] == "rotary":
        t = case["tokens"]
        pages = _pages(case, t) + 8
        state.update(
            q=normal(t, case["heads_q"], DIM), k=normal(t, case["heads_kv"], DIM),
            v=normal(t, case["heads_kv"], DIM),
            positions=torch.randint(0, case["far"], (t,), generator=gen, device="cuda").to(
                torch.int32),
            slots=shuffled(pages * case["page"])[:t].contiguous(),
            k_cache=torch.zeros(pages, case["page"], case["heads_kv"], DIM,
                                dtype=TYPES[case["dtype"]], device="cuda"))
        state["v_cache"] = torch.zeros_like(state["k_cache"])
        freq, factor = _frequencies(case)
        state.update(freq=freq.cuda(), factor=factor)
        if own:
            from fa_amd.serving import Rotary, RotaryConfig
            scaling = dict(scaling="by_parts", factor=8.0, original=4096) if case["scaled"] else {}
            state["own"] = Rotary(RotaryConfig(rotary_dim=case["rotary"], base=10000.0,
                                               layout=case["layout"], **scaling))
        return state
    if case["op"] == "window":
        def rows(heads, n):
            if case["layout"] == "bnhd":
                return normal(case["batch"], n, heads, DIM).transpose(1, 2)
            return normal(case["batch"], heads, n, DIM)

        state.update(q=rows(case["heads_q"], case["seq_q"]), k=rows(case["heads_kv"], case["seq_k"]),
                     v=rows(case["heads_kv"], case["seq_k"]))
        if own:
            from fa_amd.serving import WindowAttention, WindowConfig
            state["own"] = WindowAttention(WindowConfig(window=case["window"], sinks=case["sinks"]))
        return state
    past, new = _lengths(case)
    held = [_pages(case, p + n) for p, n in zip(past, new)]
    pool = shuffled(sum(held) + 5)
    table = torch.zeros(case["batch"], max(held), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = pool[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    shape = (len(pool), case["page"], case["heads_kv"], DIM)
    state.update(q=normal(starts[-1], case["heads_q"], DIM), k_cache=normal(*shape),
                 v_cache=normal(*shape), table=table, starts=_ints(starts),
                 lengths=_ints([p + n for p, n in zip(past, new)]), max_new=max(new),
                 host=(past, new, starts))
    if own:
        from fa_amd.serving import PagedAttention, PagedConfig
        state["own"] = PagedAttention(PagedConfig(window=case["window"] or None,
                                                  sinks=case["sinks"]))
    return state


def run(state):
    case, op = state["case"], state.get("own")
    if case["op"] == "plan":
        if op is None:
            return _plain_plan(state)
        plan = op(state["past"], state["new"], state["table"], state["pages"], state["taken"],
                  state["tokens"])
        return (state["table"], plan.query_starts, plan.key_lengths, plan.positions, plan.slots,
                plan.taken)
    if case["op"] == "rotary":
        if op is None:
            return _plain_rotary(state)
        q = op.append(state["q"], state["k"], state["v"], state["positions"], state["slots"],
                      state["k_cache"], state["v_cache"])
        return q, state["k_cache"], state["v_cache"]
    if case["op"] == "window":
        if op is None:
            return _plain_window(state)
        return op(state["q"], state["k"], state["v"], return_lse=case["lse"])
    if op is None:
        return _plain_paged(state)
    return op(state["q"], state["k_cache"], state["v_cache"], state["table"], state["starts"],
              state["lengths"], state["max_new"], return_lse=case["lse"])


# The plain forms.

def _plain_plan(state):
    page, tokens = state["case"]["page"], state["tokens"]
    past, new, table = state["past"].long(), state["new"].long(), state["table"]
    batch = len(past)
    zero = past.new_zeros(1)
    starts = torch.cat([zero, new.cumsum(0)])
    held, full = (past + page - 1) // page, (past + new + page - 1) // page
    need = torch.cat([zero, (full - held).cumsum(0)])
    first = state["taken"].long() + need[:-1]
    column = torch.arange(table.shape[1], device=table.device)
    fresh = (column >= held[:, None]) & (column < full[:, None])
    source = (first[:, None] + column - held[:, None]).clamp(0, len(state["pages"]) - 1)
    table.copy_(torch.where(fresh, state["pages"][source], table))
    token = torch.arange(tokens, device=table.device)
    ends = torch.zeros(tokens + 1, dtype=torch.int64, device=table.device)
    ends.index_add_(0, starts[1:].clamp(max=tokens), torch.ones_like(past))
    request = ends.cumsum(0)[:tokens]
    inside = request < batch
    request = request.clamp(max=batch - 1)
    position = torch.where(inside, past[request] + token - starts[request], 0)
    slot = table[request, (position // page).clamp(max=table.shape[1] - 1)].long() * page + \
        position % page
    slot = torch.where(inside, slot, -1)
    return (table, starts.int(), (past + new).int(), position.int(), slot.int(),
            (state["taken"].long() + need[-1:]).int())


def _turn(x, cos, sin, rotary, layout):
    x = x.float()
    out = x.clone()
    if layout == "half":
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        out[..., :rotary // 2] = a * cos - b * sin
        out[..., rotary // 2:rotary] = b * cos + a * sin
    else:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        out[..., 0:rotary:2] = a * cos - b * sin
        out[..., 1:rotary:2] = b * cos + a * sin
    return out


def _plain_rotary(state):
    case = state["case"]
    angle = state["positions"].double()[:, None, None] * state["freq"]
    cos = (angle.cos() * state["factor"]).float()
    sin = (angle.sin() * state["factor"]).float()
    q = _turn(state["q"], cos, sin, case["rotary"], case["layout"])
    k = _turn(state["k"], cos, sin, case["rotary"], case["layout"])
    k_cache, v_cache, slots = state["k_cache"], state["v_cache"], state["slots"].long()
    k_cache.view(-1, *k.shape[1:])[slots] = k.to(k_cache.dtype)
    v_cache.view(-1, *k.shape[1:])[slots] = state["v"]
    return q.to(state["q"].dtype), k_cache, v_cache


def _attend(q, k, v, position, key, window, sinks):
    """Rows q [G, R, 128] of one KV head's group at positions [R] over keys
    [N, 128] at positions ``key``: the result and the log-sum-exp, in 32 bits."""
    group, rows, _ = q.shape
    s = torch.mm(q.float().reshape(group * rows, DIM).contiguous(),
                 k.float().t().contiguous()).view(group, rows, -1) * DIM ** -0.5
    hidden = key > position[:, None]
    if window:
        hidden |= (key <= position[:, None] - window) & (key >= sinks)
    s.masked_fill_(hidden, float("-inf"))
    top = s.amax(-1, keepdim=True)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.mm(s.view(group * rows, -1), v.float()).view(group, rows, DIM) / total
    return o, (total.log() + top).squeeze(-1)


def _seen(first, last, window, sinks):
    """Keys that rows at positions first..last see at most: [0, a) and [b, last]."""
    b = max(0, first - window + 1) if window else 0
    return min(sinks, b) if window else 0, b


ROWS = 1024                # rows of a plain product


def _plain_window(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    group, window, sinks = case["heads_q"] // case["heads_kv"], case["window"], case["sinks"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    past = case["seq_k"] - case["seq_q"]
    for b in range(case["batch"]):
        for h in range(case["heads_kv"]):
            heads = slice(h * group, (h + 1) * group)
            for r0 in range(0, case["seq_q"], ROWS):
                r1 = min(case["seq_q"], r0 + ROWS)
                a, lo = _seen(past + r0, past + r1 - 1, window, sinks)
                hi = past + r1
                position = torch.arange(past + r0, hi, device=q.device)
                key = torch.cat([torch.arange(a, device=q.device),
                                 torch.arange(lo, hi, device=q.device)])
                o, l = _attend(q[b, heads, r0:r1], k[b, h, key], v[b, h, key], position, key, window,
                               sinks)
                out[b, heads, r0:r1] = o.to(out.dtype)
                lse[b, heads, r0:r1] = l
    return (out, lse) if case["lse"] else out


def _plain_paged(state):
    case = state["case"]
    q, table, page = state["q"], state["table"], case["page"]
    group, window, sinks = case["heads_q"] // case["heads_kv"], case["window"], case["sinks"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    past, new, starts = state["host"]
    for b in range(case["batch"]):
        for r0 in range(0, new[b], ROWS):
            r1 = min(new[b], r0 + ROWS)
            a, lo = _seen(past[b] + r0, past[b] + r1 - 1, window, sinks)
            hi = past[b] + r1
            position = torch.arange(past[b] + r0, hi, device=q.device)
            key = torch.cat([torch.arange(a, device=q.device), torch.arange(lo, hi, device=q.device)])
            where = table[b, key // page].long(), key % page
            rows = slice(starts[b] + r0, starts[b] + r1)
            k, v = state["k_cache"][where], state["v_cache"][where]
            for h in range(case["heads_kv"]):
                heads = slice(h * group, (h + 1) * group)
                o, l = _attend(q[rows, heads].transpose(0, 1), k[:, h], v[:, h], position, key,
                               window, sinks)
                out[rows, heads] = o.transpose(0, 1).to(out.dtype)
                lse[rows, heads] = l.t()
    return (out, lse) if case["lse"] else out


def _pairs(past, new, window, sinks):
    """(row, key) pairs that rows at positions past .. past + new - 1 see."""
    total = sum(range(past + 1, past + new + 1)) if not window else 0
    if window:
        for p in range(past, past + new):
            total += min(p + 1, window + min(sinks, max(0, p + 1 - window)))
    return total


def work(case):
    """What a call cannot do without: inputs read once, outputs written once."""
    if case["op"] == "plan":
        past, new = _lengths(case)
        pages = sum(_pages(case, p + n) - _pages(case, p) for p, n in zip(past, new))
        return {"bytes": 16 * case["batch"] + 8 * (sum(new) + case["slack"]) + 8 * pages + 12,
                "flops": 0}
    if case["op"] == "rotary":
        rows = case["tokens"]
        elements = rows * DIM * (case["heads_q"] + 2 * case["heads_kv"])
        turned = rows * case["rotary"] * (case["heads_q"] + case["heads_kv"])
        return {"bytes": 2 * 2 * elements + 8 * rows + 4 * case["rotary"], "flops": 3 * turned}
    if case["op"] == "window":
        past, new = [case["seq_k"] - case["seq_q"]] * case["batch"], [case["seq_q"]] * case["batch"]
        entries = 0
    else:
        past, new = _lengths(case)
        entries = 4 * sum(_pages(case, p + n) for p, n in zip(past, new))
    keys = pairs = 0
    for p, n in zip(past, new):
        a, lo = _seen(p, p + n - 1, case["window"], case["sinks"])
        keys += a + p + n - lo
        pairs += _pairs(p, n, case["window"], case["sinks"])
    rows = sum(new) * case["heads_q"]
    return {"bytes": 2 * 2 * rows * DIM + 2 * 2 * keys * case["heads_kv"] * DIM + entries +
            (4 * rows if case["lse"] else 0),
            "flops": 4 * DIM * case["heads_q"] * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(state)
    if case["op"] == "rotary":
        return _exact_rotary(state)
    window = case["window"] or 1 << 40
    group = case["heads_q"] // case["heads_kv"]
    q = state["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(q.shape[:-1], dtype=torch.float64, device="cuda")
    if case["op"] == "window":
        past, new = [case["seq_k"] - case["seq_q"]] * case["batch"], [case["seq_q"]] * case["batch"]
    else:
        past, new, starts = state["host"]
    for b, (p, n) in enumerate(zip(past, new)):
        if case["op"] == "paged":
            ids = state["table"][b, :_pages(case, p + n)].long()
            stored = [c[ids].flatten(0, 1)[:p + n].transpose(0, 1)
                      for c in (state["k_cache"], state["v_cache"])]
        else:
            stored = [state["k"][b], state["v"][b]]
        for hq in range(case["heads_q"]):
            keys, values = (t[hq // group].double().contiguous() for t in stored)
            for i in range(0, n, 512):
                m = min(512, n - i)
                if case["op"] == "paged":
                    x = q[starts[b] + i:starts[b] + i + m, hq]
                else:
                    x = q[b, hq, i:i + m]
                # Every key's score; the mask, not a slice, leaves keys out.
                lo = max(0, p + i - window + 1) if case["sinks"] == 0 else 0
                s = x.double() @ keys[lo:p + i + m].t() / math.sqrt(DIM)
                row = torch.arange(p + i, p + i + m, device="cuda")[:, None]
                col = torch.arange(lo, p + i + m, device="cuda")[None]
                visible = (col <= row) & ((row - col < window) | (col < case["sinks"]))
                s = torch.where(visible, s, -math.inf)
                total = torch.logsumexp(s, dim=1)
                o = torch.exp(s - total[:, None]) @ values[lo:p + i + m]
                if case["op"] == "paged":
                    out[starts[b] + i:starts[b] + i + m, hq] = o
                    lse[starts[b] + i:starts[b] + i + m, hq] = total
                else:
                    out[b, hq, i:i + m] = o
                    lse[b, hq, i:i + m] = total
    return (out, lse) if case["lse"] else out


def _exact_plan(state):
    page, pages = state["case"]["page"], state["pages"].tolist()
    table = state["table"].tolist()
    at = state["taken"].item()
    starts, lengths, positions, slots = [0], [], [], []
    for row, past, new in zip(table, state["past"].tolist(), state["new"].tolist()):
        for column in range((past + page - 1) // page, (past + new + page - 1) // page):
            row[column] = pages[at]
            at += 1
        for position in range(past, past + new):
            positions.append(position)
            slots.append(row[position // page] * page + position % page)
        starts.append(starts[-1] + new)
        lengths.append(past + new)
    rest = state["tokens"] - len(slots)
    return tuple(_ints(x) for x in (table, starts, lengths, positions + [0] * rest,
                                    slots + [-1] * rest, [at]))


def _exact_rotary(state):
    """As a product of complex numbers of 64-bit parts."""
    case = state["case"]
    rotary = case["rotary"]
    angle = state["positions"].double()[:, None] * state["freq"][None]
    turn = torch.polar(torch.full_like(angle, state["factor"]), angle)[:, None]

    def turned(x):
        x = x.double()
        pairs = x[..., :rotary]
        if case["layout"] == "half":
            pairs = pairs.unflatten(-1, (2, rotary // 2)).transpose(-1, -2)
        else:
            pairs = pairs.unflatten(-1, (rotary // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if case["layout"] == "half":
            z = z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., rotary:]], -1)

    caches = []
    for x in (turned(state["k"]), state["v"].double()):
        cache = torch.zeros(state["k_cache"].shape, dtype=torch.float64, device="cuda")
        cache[state["slots"].long() // case["page"], state["slots"].long() % case["page"]] = x
        caches.append(cache)
    return (turned(state["q"]), *caches)
