"""Paged attention against the plain 64-bit form: lengths from one token on, odd
sizes, pages, strides, windows and sinks, empty rows, hidden NaN, bad pages,
streams and captures."""

import random

import pytest
import torch

from fa_amd.serving import PagedAttention, PagedConfig

from serving_reference import paged64
from test_gpu_parity import say

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lib():
    from fa_amd import serving

    return serving.load_library()


class Batch:
    """Requests with (earlier, new) tokens, their pages anywhere in a cache whose
    other rows hold `filler`."""

    def __init__(self, spans, heads=(12, 1), page=16, dtype="fp16", seed=0, layout="tokens",
                 filler=float("nan"), pad_rows=0, spare=3):
        rng = random.Random(seed)
        torch.manual_seed(seed)
        self.spans, self.page = spans, page
        heads_q, heads_kv = heads
        held = [-(-(p + n) // page) for p, n in spans]
        ids = list(range(sum(held) + spare))
        rng.shuffle(ids)
        width = max(held + [1])
        self.table, at = [], 0
        for n in held:
            self.table.append(ids[at:at + n] + [-1 - rng.randint(0, 5)] * (width - n))
            at += n
        self.lengths = [p + n for p, n in spans]
        self.starts = [0]
        for _, n in spans:
            self.starts.append(self.starts[-1] + n)
        shape = (len(ids), page, heads_kv, 128)
        dtype = TYPES[dtype]
        self.k, self.v = (torch.full(shape, filler, dtype=dtype) for _ in range(2))
        for row, length in zip(self.table, self.lengths):
            for j in range(-(-length // page)):
                n = min(page, length - j * page)
                self.k[row[j], :n] = torch.randn(n, heads_kv, 128).to(dtype)
                self.v[row[j], :n] = torch.randn(n, heads_kv, 128).to(dtype)
        self.q = torch.randn(self.starts[-1] + pad_rows, heads_q, 128).to(dtype)
        self.layout = layout

    def gpu(self):
        def stored(c):
            if self.layout == "heads":           # [pages, heads, tokens, 128]
                return c.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            if self.layout == "pair":            # k and v of a page side by side
                both = torch.stack([self.k, self.v], 1).cuda()
                return both[:, 0] if c is self.k else both[:, 1]
            return c.cuda()

        q = self.q.cuda()
        if self.layout == "heads":
            q = q.transpose(0, 1).contiguous().transpose(0, 1)
        return (q, stored(self.k), stored(self.v), torch.tensor(self.table, dtype=torch.int32).cuda(),
                torch.tensor(self.starts, dtype=torch.int32).cuda(),
                torch.tensor(self.lengths, dtype=torch.int32).cuda(), max(n for _, n in self.spans))

    def check(self, o, lse, window=None, sinks=0, scale=None):
        want, want_lse, tol, tol_lse = paged64(self.q, self.k, self.v, self.table, self.starts,
                                               self.lengths, window, sinks, scale)
        n = self.starts[-1]
        compare(o[:n].cpu(), want[:n], tol[:n])
        if lse is not None:
            compare(lse[:n].cpu(), want_lse[:n], tol_lse[:n])


def compare(got, want, tol):
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    bad = ~same & ~(want.isfinite() & (off <= tol))
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, first at "
                           f"{bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]} +- {tol[bad][0]}")


def run(batch, lib, window=None, sinks=0, **kw):
    op = PagedAttention(PagedConfig(window=window, sinks=sinks), lib)
    say(f"case paged {batch.spans[:6]} page {batch.page} q {tuple(batch.q.shape)} kv {batch.k.shape[2]} "
        f"{batch.q.dtype} window {window} sinks {sinks} {batch.layout}")
    o, lse = op(*batch.gpu(), return_lse=True, **kw)
    torch.cuda.synchronize()
    return o, lse


# Decode and a few rows: (spans, heads, page, dtype)
FEW = [
    ([(0, 1)], (12, 1), 16, "fp16"),
    ([(4, 1)], (1, 1), 16, "bf16"),
    ([(15, 1), (16, 1), (17, 1)], (8, 1), 16, "fp16"),
    ([(126, 1), (127, 1), (128, 1)], (12, 1), 64, "bf16"),
    ([(4098, 1)], (12, 1), 16, "fp16"),
    ([(700, 1), (0, 1), (2049, 1), (33, 1), (1, 1)], (64, 8), 32, "bf16"),
    ([(20000, 1)], (8, 1), 256, "fp16"),
    ([(300, 2), (511, 5), (0, 3)], (12, 1), 16, "fp16"),
    ([(300, 4), (0, 0), (90, 1), (0, 0)], (16, 16), 128, "bf16"),
    ([(1000, 1)] * 70, (4, 2), 64, "fp16"),
    ([(37, 1)], (24, 3), 1024, "bf16"),
]
# Prompts and chunks.
MANY = [
    ([(0, 300)], (12, 1), 16, "fp16"),
    ([(0, 65)], (1, 1), 16, "bf16"),
    ([(1000, 257)], (4, 4), 64, "fp16"),
    ([(77, 700)], (8, 2), 128, "bf16"),
    ([(5000, 33)], (12, 1), 32, "fp16"),
    ([(0, 129), (300, 1), (250, 80), (1, 1), (0, 0), (40, 64)], (32, 8), 16, "bf16"),
    ([(3, 1500)], (24, 2), 256, "fp16"),
    ([(511, 128), (0, 1)], (3, 3), 16, "fp16"),
    ([(60, 400), (400, 60), (130, 130)], (64, 8), 64, "fp16"),
]


@pytest.mark.parametrize("spans,heads,page,dtype", FEW + MANY)
def test_against_64_bits(lib, spans, heads, page, dtype):
    batch = Batch(spans, heads, page, dtype)
    batch.check(*run(batch, lib))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 3), (128, 4), (129, 0), (500, 200), (10 ** 9, 7)])
@pytest.mark.parametrize("spans,heads,page,dtype", [
    ([(700, 1), (0, 1), (2049, 1), (33, 2)], (64, 8), 32, "fp16"),
    ([(1000, 257), (90, 1)], (4, 4), 64, "bf16"),
    ([(0, 900)], (12, 1), 16, "fp16"),
])
def test_window_and_sinks(lib, spans, heads, page, dtype, window, sinks):
    batch = Batch(spans, heads, page, dtype, seed=window % 1000)
    batch.check(*run(batch, lib, window, sinks), window, sinks)


@pytest.mark.parametrize("layout", ["heads", "pair"])
@pytest.mark.parametrize("spans", [[(300, 1), (9, 1)], [(100, 200), (5, 1)]])
def test_layouts(lib, layout, spans):
    batch = Batch(spans, (8, 2), 32, "bf16", seed=5, layout=layout)
    batch.check(*run(batch, lib, scale=0.2), scale=0.2)
