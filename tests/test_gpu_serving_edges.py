"""The serving operators where they go wrong most easily: NaN and infinities in
hidden places, bad pages and lengths, padded batches, caches past 32-bit offsets,
streams, captured graphs, repeated calls, random small cases."""

import random

import pytest
import torch

from fa_amd.cache import CacheConfig, PagedCache
from fa_amd.serving import (PagedAttention, PagedConfig, PagePlanner, Rotary, RotaryConfig,
                            WindowAttention, WindowConfig)

from serving_reference import attend64, bounds, paged64, plan, rotate64
from test_gpu_paged import FEW, MANY, Batch, compare, run
from test_gpu_parity import say
from test_gpu_rotary import bound as rotary_bound
from test_gpu_window import check as check_window
from test_gpu_window import tensors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from fa_amd import serving

    return serving.load_library()


# NaN and infinities.

HIDDEN = [([(700, 3)], (12, 1), 16), ([(0, 300)], (12, 1), 16), ([(300, 130), (7, 1)], (4, 2), 64),
          ([(20, 90)], (1, 1), 32)]


@pytest.mark.parametrize("spans,heads,page", HIDDEN)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_bad_new_token_reaches_only_later_rows(lib, spans, heads, page, value, dtype):
    # One new token in the middle of a chunk has a bad K or V, in one dim of one
    # head or in all: rows before it are as if it were not there, rows after it get
    # what the formula gives.
    for where in ("k", "v", "v one dim"):
        batch = Batch(spans, heads, page, dtype, seed=7)
        past, new = spans[0]
        at = past + new // 2
        slot = batch.table[0][at // page], at % page
        if where == "k":
            # In dim 0, where q is positive: an infinite score of one sign.
            batch.k[slot][0, 0] = value
            batch.q[..., 0] = batch.q[..., 0].abs() + 0.1
        elif where == "v":
            batch.v[slot] = value
        else:
            batch.v[slot][0, 5] = value
        o, lse = run(batch, lib)
        check_values(batch, o, lse)


def check_values(batch, o, lse, window=None, sinks=0):
    """Against the formula key by key. A row with an infinite score has NaN for its
    log-sum-exp as for its values (infinity minus infinity)."""
    want, want_lse, tol, tol_lse = paged64(batch.q, batch.k, batch.v, batch.table, batch.starts, batch.lengths,
                                           window, sinks)
    want_lse = torch.where(want_lse == float("inf"), float("nan"), want_lse)
    n = batch.starts[-1]
    compare(o[:n].cpu(), want[:n], tol[:n])
    compare(lse[:n].cpu(), want_lse[:n], tol_lse[:n])


@pytest.mark.parametrize("spans,heads,page", HIDDEN)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_infinities_beside_a_hidden_nan(lib, spans, heads, page, dtype):
    # A dim with NaN at the newest key and infinities at older ones: rows before it
    # keep the infinity of what they see, and NaN where they see both signs.
    inf = float("inf")
    batch = Batch(spans, heads, page, dtype, seed=9)
    past, new = spans[0]
    last, first = past + new - 1, min(5, past + new - 2)
    at = lambda key: (batch.table[0][key // page], key % page)
    batch.v[at(last)] = float("nan")
    batch.v[at(first)][..., 0:2] = inf
    batch.v[at(first)][..., 8] = inf
    batch.v[at(first + 1)][..., 8] = -inf
    batch.v[at(first + 1)][..., 9] = -inf
    o, lse = run(batch, lib)
    check_values(batch, o, lse)


@pytest.mark.parametrize("spans,heads,page", HIDDEN + [([(30000, 200), (30000, 2)], (8, 1), 32)])
def test_values_of_nan_alone(lib, spans, heads, page):
    batch = Batch(spans, heads, page, "fp16", seed=10)
    batch.v[:] = float("nan")
    o, lse = run(batch, lib)
    check_values(batch, o, lse)


@pytest.mark.parametrize("spans,heads,page", HIDDEN)
@pytest.mark.parametrize("window,sinks", [(40, 0), (40, 3)])
def test_nan_outside_the_window(lib, spans, heads, page, window, sinks):
    batch = Batch(spans, heads, page, "fp16", seed=8)
    past, new = spans[0]
    # A key that the first rows still see and the last do not, or that none sees.
    for at in {max(0, past - window + 5), sinks + 1 if past > window + sinks + 2 else max(0, past - 1)}:
        batch.v[batch.table[0][at // page], at % page] = float("nan")
        batch.k[batch.table[0][at // page], at % page, 0, 3] = float("nan")
    o, lse = run(batch, lib, window, sinks)
    check_values(batch, o, lse, window, sinks)


def test_window_form_keeps_hidden_nan_out(lib):
    q, k, v = tensors(1, 4, 2, 200, 300, "bf16", seed=3)
    k[0, 1, 150], v[0, 0, 220], v[0, 1, 290, 7] = float("nan"), float("nan"), float("inf")
    check_window(lib, q, k, v, window=60, sinks=2)


@pytest.mark.parametrize("spans", [[(900, 1)], [(100, 120)]])
def test_a_nan_query_row_is_nan_alone(lib, spans):
    batch = Batch(spans, (12, 1), 16, "fp16", seed=9)
    batch.q[0, 3, 5] = float("nan")
    o, lse = run(batch, lib)
    check_values(batch, o, lse)
    assert o[0, 3].isnan().all() and lse[0, 3].isnan() and not o[0, 2].isnan().any()


@pytest.mark.parametrize("new", [1, 200])
def test_scores_far_below_zero(lib, new):
    # Scores of about -1.1e6, all equal.
    batch = Batch([(150, new)], (4, 1), 16, "bf16", seed=10)
    batch.k[:] = torch.where(batch.k.isnan(), batch.k, torch.full_like(batch.k, -100.0))
    batch.q[:] = 1000.0
    o, lse = run(batch, lib)
    # The mean of the values, to the rounding of P, the same for all keys, and of the
    # result (2^-8 of it each), and the FP32 sums.
    for i in (0, new - 1):
        n = 150 + i + 1
        key = torch.arange(n)
        v = batch.v[torch.tensor(batch.table[0])[key // 16].long(), key % 16, 0].double()
        want = v.mean(0)
        tol = 2.01 * 2.0 ** -8 * want.abs() + 2.0 ** -18 * v.abs().mean(0)
        compare(o[i, 0].cpu(), want, tol)
    assert torch.isfinite(lse).all() and (lse < -1e6).all()


@pytest.mark.parametrize("spans,heads", [([(100000, 1)], (12, 1)), ([(100000, 1)] * 3, (4, 2)),
                                         ([(20000, 130)], (2, 1))])
def test_a_nan_score_in_one_of_many_pieces(lib, spans, heads):
    # The joins: a piece whose log-sum-exp is NaN among hundreds of others.
    batch = Batch(spans, heads, 64, "bf16", seed=11)
    at = spans[0][0] * 3 // 4
    batch.k[batch.table[0][at // 64], at % 64, 0] = float("nan")
    o, lse = run(batch, lib)
    check_values(batch, o, lse)
    own = slice(0, spans[0][1]), slice(0, heads[0] // heads[1])
    assert o[own].isnan().all() and lse[own].isnan().all()


# Which kernel, how many pieces.

@pytest.mark.parametrize("keys", [8192, 8193, 32768, 32769, 131072])
@pytest.mark.parametrize("heads", [(12, 1), (31, 1)])
def test_joins_of_every_size(lib, keys, heads):
    # One request: 32, 33, 128, 129 and 512 shares.
    batch = Batch([(keys - 1, 1)], heads, 256, "fp16", seed=12)
    o, lse = run(batch, lib)
    batch.check(o, lse)


@pytest.mark.parametrize("requests", [3, 11])
@pytest.mark.parametrize("longest", [8, 9])
def test_two_row_tiles_a_request(lib, requests, longest):
    # Up to 64 rows a KV head, and 72, in launches of few and of more row tiles.
    spans = [(150 + 97 * i, 1 + (longest - 1) * (i % 3) // 2) for i in range(requests)]
    batch = Batch(spans, (64, 8), 32, "bf16", seed=13)
    o, lse = run(batch, lib)
    batch.check(o, lse)


# Lengths, tables, padding.

def test_rows_without_keys_and_empty_requests(lib):
    # More new rows than tokens: the first rows stand before the first token. One
    # request without tokens, one without rows.
    batch = Batch([(20, 4), (0, 9), (33, 0), (0, 40)], (12, 1), 16, "fp16")
    batch.lengths[1], batch.lengths[3] = 4, 0
    o, lse = run(batch, lib)
    batch.check(o, lse)
    assert (o[4:9] == 0).all() and (lse[4:9] == -float("inf")).all() and (o[13:53] == 0).all()


@pytest.mark.parametrize("heads", [(12, 1), (64, 8)])
def test_rows_behind_the_last_request_stay(lib, heads):
    for spans in ([(300, 1), (20, 1)], [(90, 150), (5, 1)]):
        batch = Batch(spans, heads, 16, "bf16", pad_rows=37)
        op = PagedAttention(library=lib)
        args = batch.gpu()
        out = torch.full_like(args[0], 3.5)
        assert op(*args, out=out) is out
        batch.check(out, None)
        assert (out[batch.starts[-1]:] == 3.5).all()


@pytest.mark.parametrize("spans,heads,page,dtype", [FEW[5], FEW[7], MANY[0], MANY[5]])
@pytest.mark.parametrize("max_new", [1, 20, 100000])
def test_max_new_only_chooses(lib, spans, heads, page, dtype, max_new):
    batch = Batch(spans, heads, page, dtype)
    say(f"case max_new {max_new} {spans}")
    o, lse = PagedAttention(library=lib)(*batch.gpu()[:6], max_new, return_lse=True)
    batch.check(o, lse)


@pytest.mark.parametrize("spans", [[(100, 1), (700, 1), (50, 1)], [(100, 200), (700, 130), (50, 1)]])
@pytest.mark.parametrize("page_id", [-1, 10 ** 6, 2 ** 31 - 1])
def test_a_page_outside_the_cache_is_loud(lib, spans, page_id):
    batch = Batch(spans, (8, 2), 16, "fp16")
    batch.table[1][4] = page_id
    o, lse = run(batch, lib)
    s = batch.starts
    assert o[s[1]:s[2]].isnan().all() and lse[s[1]:s[2]].isnan().all()
    batch.table[1] = list(batch.table[0])        # any valid pages, for the reference
    want, want_lse, tol, tol_lse = paged64(batch.q, batch.k, batch.v, batch.table, s, [batch.lengths[0], 1, batch.lengths[2]])
    for b in (0, 2):
        rows = slice(s[b], s[b + 1])
        compare(o[rows].cpu(), want[rows], tol[rows])
        compare(lse[rows].cpu(), want_lse[rows], tol_lse[rows])


@pytest.mark.parametrize("spans", [[(100, 1), (700, 1)], [(100, 200), (700, 130)]])
def test_a_request_longer_than_its_table_is_loud(lib, spans):
    batch = Batch(spans, (8, 2), 16, "fp16")
    args = list(batch.gpu())
    op = PagedAttention(library=lib)
    for length in (16 * args[3].shape[1] + 1, 2 ** 31 - 1):
        args[5] = torch.tensor([batch.lengths[0], length], dtype=torch.int32).cuda()
        o = op(*args)
        torch.cuda.synchronize()
        s = batch.starts
        assert o[s[1]:].isnan().all() and not o[:s[1]].isnan().any()


def test_starts_and_lengths_out_of_range_stay_in_bounds(lib):
    # Nothing to compare with: such a call writes no row but its own and returns.
    batch = Batch([(100, 1), (200, 40), (30, 1)], (12, 1), 16, "fp16", pad_rows=5)
    args = list(batch.gpu())
    op = PagedAttention(library=lib)
    for starts in ([-5, 3, 1, 2], [0, 10 ** 9, 5, 10 ** 9], [7, 7, 7, 7], [9, 4, 2, 0]):
        for lengths in ([-3, 0, 5], [2 ** 31 - 1, 1, -2 ** 31]):
            say(f"case starts {starts} lengths {lengths}")
            args[4] = torch.tensor(starts, dtype=torch.int32).cuda()
            args[5] = torch.tensor(lengths, dtype=torch.int32).cuda()
            op(*args)
            torch.cuda.synchronize()
    args[4:6] = batch.gpu()[4:6]
    o, lse = op(*args, return_lse=True)          # and the next call is right
    batch.check(o, lse)


def test_planner_takes_odd_lengths(lib):
    # Negative lengths count as 0; a table row that ends early and too few pages give -1.
    past, new = [-4, 5, 2 ** 31 - 1, 30], [3, -1, 7, 40]
    table = [[50 + 3 * b, 51 + 3 * b, 52 + 3 * b] for b in range(4)]
    on = torch.tensor(table, dtype=torch.int32).cuda()
    got = PagePlanner(16, lib)(torch.tensor(past, dtype=torch.int32).cuda(), torch.tensor(new, dtype=torch.int32).cuda(),
                               on, torch.arange(2, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda(), 60)
    assert got.query_starts.tolist() == [0, 3, 3, 10, 50]
    assert got.key_lengths.tolist() == [3, 5, 2 ** 31 - 1, 70]
    slots = got.slots.tolist()
    assert slots[:3] == [0, 1, 2] and slots[3:10] == [-1] * 7
    # Request 2 took the last free page; request 3 has two tokens in its second page, no
    # page for the next 16, and no table entry for the rest.
    assert slots[10:12] == [60 * 16 + 14, 60 * 16 + 15] and slots[12:] == [-1] * 48
    assert on[3].tolist() == [59, 60, -1] and on[0].tolist() == [0, 51, 52] and got.taken.tolist() == [5]


@pytest.mark.parametrize("batch,chunks", [(300, 0), (700, 0), (1100, 3), (4096, 0), (2000, 2000)])
def test_many_requests(lib, batch, chunks):
    # More requests than a workgroup has threads; chunks of 33 and more rows at
    # both ends and in the middle.
    rng = random.Random(batch)
    spans = [(rng.randint(0, 40), 1) for _ in range(batch)]
    for i in ([0, batch // 2, batch - 1] if chunks == 3 else range(chunks)):
        spans[i] = (rng.randint(0, 20), rng.randint(33, 36))
    batch = Batch(spans, (2, 1), 16, "bf16", seed=batch)
    batch.check(*run(batch, lib))


# Large offsets and strides.

def test_a_cache_past_32_bit_offsets(lib):
    # 5.4 GB each of K and V, the request's pages at both ends; rows behind its last
    # key hold NaN.
    heads_q, heads_kv, page, pages = 16, 8, 256, 10300
    k = torch.empty(pages, page, heads_kv, 128, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    ids = [pages - 1, 0, pages - 2, 8191, 8192, 5]
    torch.manual_seed(0)
    for new in (1, 40):
        length = 5 * page + 77
        for c in (k, v):
            for i in ids:
                c[i] = torch.randn(page, heads_kv, 128, device="cuda").half()
            c[ids[5], 77:] = float("nan")
        q = torch.randn(new, heads_q, 128, device="cuda").half()
        say(f"case far pages, {new} rows")
        o, lse = PagedAttention(library=lib)(q, k, v, torch.tensor([ids], dtype=torch.int32).cuda(),
                                             torch.tensor([0, new], dtype=torch.int32).cuda(),
                                             torch.tensor([length], dtype=torch.int32).cuda(), new, return_lse=True)
        at = torch.tensor(ids)
        want, want_lse, tol, tol_lse = paged64(q.cpu(), k[at.cuda()].cpu(), v[at.cuda()].cpu(), [list(range(6))], [0, new],
                                               [length])
        compare(o.cpu(), want, tol)
        compare(lse.cpu(), want_lse, tol_lse)
    # And stored there.
    slots = torch.tensor([pages * page - 1, 3, (pages - 1) * page], dtype=torch.int32).cuda()
    kv = torch.randn(3, heads_kv, 128, device="cuda").half()
    positions = torch.tensor([5, 70000, 0], dtype=torch.int32).cuda()
    config = RotaryConfig()
    Rotary(config, lib).append(torch.randn(3, heads_q, 128, device="cuda").half(), kv, kv, positions, slots, k, v)
    turned = rotate64(kv.cpu(), positions.cpu(), config.frequencies(), 1.0, "half")
    for i, slot in enumerate(slots.tolist()):
        assert torch.equal(v[slot // page, slot % page], kv[i])
        compare(k[slot // page, slot % page].cpu(), turned[i], rotary_bound(kv.cpu(), turned, config)[i])


def test_a_contiguous_tensor_past_32_bit_offsets(lib):
    # Keys 64 KiB apart (one head of many side by side), 5 GB of them.
    base = torch.empty(80000, 256, 128, dtype=torch.float16, device="cuda")
    k, v = base[:, 3].unsqueeze(0).unsqueeze(0), base[:, 250].unsqueeze(0).unsqueeze(0)
    torch.manual_seed(1)
    for nq in (2, 100):
        base[-1000:, 3] = torch.randn(1000, 128, device="cuda").half()
        base[-1000:, 250] = torch.randn(1000, 128, device="cuda").half()
        q = torch.randn(1, 4, nq, 128, device="cuda").half()
        say(f"case far rows, {nq}")
        o = WindowAttention(WindowConfig(window=700), lib)(q, k, v)
        pos, key = torch.arange(80000 - nq, 80000), torch.arange(79000, 80000)
        for h in range(4):
            x = attend64(q[0, h].cpu(), k[0, 0, -1000:].cpu(), v[0, 0, -1000:].cpu(), pos, key, 700, 0, 128 ** -0.5)
            compare(o[0, h].cpu(), x[0], bounds(torch.float16, *x, 1000)[0])


def test_a_long_request(lib):
    batch = Batch([(131071, 1), (70, 1)], (4, 1), 64, "bf16")
    batch.check(*run(batch, lib))


# Streams, graphs, repetition.

def test_repeated_calls_are_the_same(lib):
    for spans in ([(3000, 1), (70, 1), (900, 1)], [(4000, 300), (50, 1)]):
        batch = Batch(spans, (12, 1), 16, "fp16")
        op = PagedAttention(library=lib)
        args = batch.gpu()
        first = [t.clone() for t in op(*args, return_lse=True)]
        for _ in range(5):
            again = op(*args, return_lse=True)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_two_streams_at_once(lib):
    op = PagedAttention(library=lib)
    batches = [Batch([(5000, 1), (900, 1)], (12, 1), 16, "fp16", seed=1), Batch([(3000, 300), (60, 1)], (8, 2), 64, "bf16", seed=2)]
    args = [b.gpu() for b in batches]
    alone = [op(*a, return_lse=True) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                results.append(op(*a, return_lse=True))
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(results):
        assert torch.equal(o, alone[i % 2][0]) and torch.equal(lse, alone[i % 2][1])


def test_inputs_of_another_stream_are_held(lib):
    # The caller drops its tensors right after the call; memory that another stream
    # allocates meanwhile must not be theirs.
    op = WindowAttention(WindowConfig(window=2000), lib)
    q, k, v = (torch.randn(4, h, 4000, 128, device="cuda").half() for h in (8, 2, 2))
    want = op(q, k, v)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        a, b, c = q.clone(), k.clone(), v.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = op(a, b, c)
        del a, b, c
        junk = [torch.full_like(t, float("nan")) for t in (q, k, v)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del junk


def test_two_captured_graphs_of_one_operator(lib):
    op = PagedAttention(PagedConfig(window=1000, sinks=4), lib)
    batches = [Batch([(5000, 1), (900, 1)], (12, 1), 16, "fp16", seed=3), Batch([(3000, 300), (60, 1)], (12, 1), 16, "fp16", seed=4)]
    args = [b.gpu() for b in batches]
    graphs, outs = [], []
    for a in args:
        op(*a)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(op(*a, return_lse=True))
        graphs.append(graph)
    for i in range(4):
        for a in args:
            a[0].copy_(torch.randn_like(a[0]))
        want = [[t.clone() for t in op(*a, return_lse=True)] for a in args]
        torch.cuda.synchronize()
        for g in (graphs if i % 2 else reversed(graphs)):
            g.replay()
        op(*args[i % 2])                         # eager work beside them
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(got, w)), i


def test_a_captured_step(lib):
    # A whole step, page plan and lengths included: each replay appends one token.
    config = CacheConfig(layers=1, heads_q=12, heads_kv=1, pages=200, page_size=16, max_batch=6, max_length=400)
    eager, captured = PagedCache(config), PagedCache(config)
    torch.manual_seed(5)
    prompt = torch.tensor([30, 16, 1, 0, 200, 77], dtype=torch.int32).cuda()
    one = torch.tensor([1, 1, 1, 0, 1, 1], dtype=torch.int32).cuda()
    q, k, v = (torch.randn(330, h, 128, device="cuda").half() for h in (12, 1, 1))
    for cache in (eager, captured):
        cache.begin(prompt, 330, 200)
        cache.attend(0, q, k, v)
    x = [torch.randn(8, h, 128, device="cuda").half() for h in (12, 1, 1)]

    def step(cache):
        cache.begin(one, 8, 1)
        return cache.attend(0, *x)

    kept = [t.clone() for t in (captured.lengths, captured.taken, captured.table, captured.k, captured.v)]
    step(captured)                               # sets up what a capture may not
    torch.cuda.synchronize()
    for t, was in zip((captured.lengths, captured.taken, captured.table, captured.k, captured.v), kept):
        t.copy_(was)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured)
    for i in range(20):
        for t in x:
            t.copy_(torch.randn_like(t))
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:5], want[:5]), i
        assert torch.equal(captured.lengths, eager.lengths) and torch.equal(captured.taken, eager.taken)
        assert torch.equal(captured.table, eager.table)


# Random small cases.

@pytest.mark.parametrize("seed", range(24))
def test_random_batches(lib, seed):
    rng = random.Random(seed)
    heads = rng.choice([(12, 1), (1, 1), (8, 2), (6, 6), (5, 1), (24, 3), (16, 8), (64, 8), (40, 8), (96, 1)])
    big = rng.random() < 0.5
    spans = [(rng.choice([0, 1, rng.randint(0, 60), rng.randint(0, 1500)]),
              rng.choice([0, 1, 1, 2, rng.randint(1, 12)]) if not big or rng.random() < 0.6 else rng.randint(1, 400))
             for _ in range(rng.randint(1, 9))]
    spans.append((rng.randint(0, 300), rng.randint(1, 30)))
    window = rng.choice([None, None, rng.randint(1, 40), rng.randint(1, 900)])
    sinks = rng.choice([0, rng.randint(1, 5), rng.randint(1, 300)]) if window else 0
    batch = Batch(spans, heads, rng.choice([16, 32, 64, 128, 512]), rng.choice(["fp16", "bf16"]), seed,
                  layout=rng.choice(["tokens", "heads", "pair"]))
    batch.check(*run(batch, lib, window, sinks), window, sinks)


@pytest.mark.parametrize("seed", range(12))
def test_random_windows(lib, seed):
    rng = random.Random(100 + seed)
    hq, hkv = rng.choice([(12, 1), (1, 1), (8, 2), (6, 6), (24, 3), (16, 8)])
    nq, nk = rng.choice([1, 2, 31, rng.randint(1, 700)]), rng.choice([1, 127, 128, 129, rng.randint(1, 1500)])
    check_window(lib, *tensors(rng.randint(1, 3), hq, hkv, nq, nk, rng.choice(["fp16", "bf16"]),
                               rng.choice(["bhnd", "bnhd"]), seed),
                 window=rng.choice([1, 7, rng.randint(1, 300), 2000]), sinks=rng.choice([0, 1, rng.randint(1, 200)]),
                 causal=rng.choice(["top_left", "bottom_right"]), scale=rng.choice([None, 0.03, 0.4]))


# The operators in a row.

@pytest.mark.parametrize("window,sinks,dtype,page", [(None, 0, "float16", 16), (50, 3, "bfloat16", 32)])
def test_a_cache_over_several_steps(lib, window, sinks, dtype, page):
    """Prompts in pieces, single tokens and idle requests over two layers, against
    attention in 64 bits over the tokens so far, rotated and rounded as stored; one
    request ends and its number and pages are taken again."""
    config = CacheConfig(layers=2, heads_q=4, heads_kv=2, pages=60, page_size=page, max_batch=4, max_length=400,
                         dtype=dtype, rotary=RotaryConfig(rotary_dim=64, layout="interleaved"),
                         attention=PagedConfig(window=window, sinks=sinks))
    cache = PagedCache(config)
    torch.manual_seed(4)
    kind = getattr(torch, dtype)
    lengths = [0] * 4
    rotate = config.rotary
    for step, new in enumerate([[70, 0, 5, 130], [1, 33, 40, 1], [1, 1, 1, 1], [20, 1, 0, 1], "release", [1, 1, 60, 1]]):
        if new == "release":
            cache.release(2)
            lengths[2] = 0
            continue
        tokens = sum(new) + 3
        say(f"case cache step {step} {new}")
        got = cache.begin(torch.tensor(new, dtype=torch.int32).cuda(), tokens, max(new))
        before, lengths = lengths, [a + b for a, b in zip(lengths, new)]
        assert got.key_lengths.tolist() == lengths
        held = [row[:-(-n // page)] for row, n in zip(cache.table.tolist(), lengths)]
        used = [i for row in held for i in row]
        assert len(set(used)) == len(used) and all(0 <= i < config.pages for i in used)
        positions = got.positions.cpu()
        for layer in range(2):
            q, k, v = (torch.randn(tokens, h, 128).to(kind) for h in (4, 2, 2))
            o = cache.attend(layer, q.cuda(), k.cuda(), v.cuda())
            # q and k as the attention saw them, each held to the rotation in 64 bits.
            qr = cache.rotary(q.cuda(), got.positions).cpu()
            args = (positions, rotate.frequencies(), rotate.magnitude, rotate.layout)
            want = rotate64(q, *args)
            compare(qr, want, rotary_bound(q, want, rotate))
            want, at = rotate64(k, *args), 0
            allowed = rotary_bound(k, want, rotate)
            for b, n in enumerate(new):
                rows = slice(at, at + n)
                at += n
                if not n:
                    continue
                pages = torch.tensor(held[b]).cuda()
                ks, vs = (c[layer, pages].flatten(0, 1)[:lengths[b]].cpu() for c in (cache.k, cache.v))
                compare(ks[before[b]:], want[rows], allowed[rows])
                assert torch.equal(vs[before[b]:], v[rows])
                key, pos = torch.arange(lengths[b]), torch.arange(before[b], lengths[b])
                for h in range(4):
                    x = attend64(qr[rows, h], ks[:, h // 2], vs[:, h // 2], pos, key, window, sinks, 128 ** -0.5)
                    compare(o[rows, h].cpu(), x[0], bounds(kind, *x, lengths[b])[0])


def test_out_must_not_be_what_is_read(lib):
    batch = Batch([(40, 3)], (2, 2), 16, "fp16")
    args = batch.gpu()
    with pytest.raises(ValueError, match="out"):
        PagedAttention(library=lib)(*args, out=args[0])
    q = torch.zeros(1, 2, 40, 128, dtype=torch.float16, device="cuda")
    for t in ([q, torch.zeros_like(q), torch.zeros_like(q)], [torch.zeros_like(q), q, torch.zeros_like(q)]):
        with pytest.raises(ValueError, match="out"):
            WindowAttention(WindowConfig(window=8), library=lib)(*t, out=q)


def test_a_cache_that_was_asked_for_too_much(lib):
    # 11 pages of 16 tokens for 20, 100 and 60 tokens: the last request misses two
    # pages and gets NaN; once it has ended, the others go on and its pages serve a new one.
    cache = PagedCache(CacheConfig(layers=1, heads_q=2, heads_kv=1, pages=11, page_size=16, max_batch=3,
                                   max_length=160))
    torch.manual_seed(6)

    def step(new):
        tokens = sum(new)
        q, k, v = (torch.randn(tokens, h, 128).half().cuda() for h in (2, 1, 1))
        cache.begin(torch.tensor(new, dtype=torch.int32).cuda(), tokens, max(new))
        return cache.attend(0, q, k, v)

    o = step([20, 100, 60])
    assert torch.isfinite(o[:120]).all() and o[-12:].isnan().all()
    cache.release(2)
    assert sorted(cache.pages.tolist()[int(cache.taken):]) == sorted(set(range(11)) - {
        i for row in cache.table.tolist() for i in row if i >= 0})
    assert torch.isfinite(step([1, 1, 30])).all()
