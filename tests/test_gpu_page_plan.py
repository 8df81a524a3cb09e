"""Page plans on the GPU against plain Python, exactly."""

import random

import pytest
import torch

from fa_amd.serving import PagePlanner

import serving_reference
from test_gpu_parity import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from fa_amd import serving

    return serving.load_library()


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def case(batch, page, seed, top=300, most=70, width=None, free=None, slack=0):
    rng = random.Random(seed)
    past = [rng.choice([0, 1, page - 1, page, rng.randint(0, top)]) for _ in range(batch)]
    new = [rng.choice([0, 1, 1, page, rng.randint(0, most)]) for _ in range(batch)]
    need = sum(-(-(p + n) // page) - -(-p // page) for p, n in zip(past, new))
    longest = max(-(-(p + n) // page) for p, n in zip(past, new))
    width = max(longest, 1) + 2 if width is None else width
    ids = list(range(10000))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(min(-(-p // page), width))] for p in past]
    table = [row + [-7] * (width - len(row)) for row in table]
    taken = rng.randint(0, 4)
    pages = ids[:taken + (need if free is None else free)]
    return past, new, table, pages, taken, sum(new) + slack


def check(lib, page, past, new, table, pages, taken, tokens):
    say(f"case plan {len(past)} requests, page {page}, {tokens} tokens")
    planner = PagePlanner(page, lib)
    on = ints(table)
    for _ in range(2):                          # a repeated call changes nothing
        got = planner(ints(past), ints(new), on, ints(pages), ints([taken]), tokens)
        want = serving_reference.plan(past, new, table, pages, taken, tokens, page)
        out = (on, got.query_starts, got.key_lengths, got.positions, got.slots, got.taken)
        for name, g, w in zip(("table", "starts", "lengths", "positions", "slots", "taken"), out,
                              want[:5] + ([want[5]],)):
            assert g.tolist() == w, name


@pytest.mark.parametrize("batch,page,slack", [(1, 16, 0), (1, 64, 9), (5, 16, 3), (64, 32, 0), (255, 16, 1),
                                              (256, 128, 300), (257, 16, 0), (1000, 64, 5), (4096, 256, 0)])
def test_against_plain(lib, batch, page, slack):
    for seed in range(3):
        check(lib, page, *case(batch, page, seed, slack=slack))


def test_pages_run_out_and_tokens_past_the_table(lib):
    for free in (0, 1, 5):
        check(lib, 16, *case(20, 16, free, free=free))
    check(lib, 16, *case(20, 16, 3, width=4))


def test_nothing_new(lib):
    check(lib, 16, [0, 5], [0, 0], [[1, 2], [3, 4]], [9], 0, 0)
    check(lib, 16, [0, 5], [0, 0], [[1, 2], [3, 4]], [9], 1, 7)
