"""Windowed attention on contiguous tensors against the plain 64-bit form."""

import pytest
import torch

from fa_amd.serving import WindowAttention, WindowConfig

from serving_reference import window64
from test_gpu_paged import TYPES, compare
from test_gpu_parity import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from fa_amd import serving

    return serving.load_library()


def tensors(b, hq, hkv, nq, nk, dtype, layout="bhnd", seed=0):
    torch.manual_seed(seed)

    def rand(h, n):
        t = torch.randn(b, h, n, 128).to(TYPES[dtype])
        return t if layout == "bhnd" else t.transpose(1, 2).contiguous().transpose(1, 2)

    return rand(hq, nq), rand(hkv, nk), rand(hkv, nk)


def check(lib, q, k, v, scale=None, **config):
    say(f"case window q {tuple(q.shape)} {q.stride()} k {tuple(k.shape)} {q.dtype} {config}")
    op = WindowAttention(WindowConfig(**config), lib)
    o, lse = op(q.cuda(), k.cuda(), v.cuda(), scale=scale, return_lse=True)
    torch.cuda.synchronize()
    want, want_lse, tol, tol_lse = window64(q, k, v, scale=scale, **config)
    compare(o.cpu(), want, tol)
    compare(lse.cpu(), want_lse, tol_lse)


@pytest.mark.parametrize("shape", [
    (1, 12, 1, 1, 1), (2, 64, 8, 1, 805), (1, 1, 1, 3, 130), (3, 8, 2, 2, 64), (1, 12, 1, 300, 300),
    (2, 4, 4, 257, 600), (1, 16, 8, 129, 129), (1, 24, 2, 700, 900), (1, 3, 3, 1000, 1000),
])
@pytest.mark.parametrize("window,sinks,dtype,layout", [
    (1, 0, "fp16", "bhnd"), (64, 5, "bf16", "bnhd"), (257, 0, "bf16", "bhnd"), (400, 130, "fp16", "bnhd"),
    (5000, 2, "fp16", "bhnd"),
])
def test_against_64_bits(lib, shape, window, sinks, dtype, layout):
    check(lib, *tensors(*shape, dtype, layout), window=window, sinks=sinks)


@pytest.mark.parametrize("shape", [(1, 12, 1, 40, 9), (2, 4, 2, 300, 100), (1, 1, 1, 700, 3), (1, 4, 1, 5, 2)])
@pytest.mark.parametrize("causal", ["top_left", "bottom_right"])
def test_rows_without_keys_and_rows_past_the_keys(lib, shape, causal):
    # Bottom right, more rows than keys: the first rows see nothing. Top left: the
    # last rows' windows lie past the keys, and without sinks they see nothing.
    for sinks in (0, 2):
        check(lib, *tensors(*shape, "fp16"), window=20, sinks=sinks, causal=causal)
