"""Rotary positions and their storage in pages against the plain 64-bit form.

A rotated value x0 c - x1 s is formed in FP32 and rounded once: half a step u of
the type of its own size, and 2^-24 (|x0 c| + |x1 s|) times a few roundings (the
angle's part of a turn, sine, cosine, factor, product, sum: 8 allowed)."""

import pytest
import torch

from fa_amd.serving import Rotary, RotaryConfig

from serving_reference import rotate64
from test_gpu_paged import TYPES, compare
from test_gpu_parity import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from fa_amd import serving

    return serving.load_library()


def bound(x, want, config):
    dtype = x.dtype
    half = config.rotary_dim // 2
    x = x.double().abs()
    size = x.clone()
    if config.layout == "half":
        size[..., :half] = size[..., half:2 * half] = x[..., :half] + x[..., half:2 * half]
    else:
        pair = x[..., 0:2 * half:2] + x[..., 1:2 * half:2]
        size[..., 0:2 * half:2] = size[..., 1:2 * half:2] = pair
    eps = 8 * 2.0 ** -24 * config.magnitude * size
    # The smallest FP16 step is 2^-24: half of it where the value is a subnormal.
    u = torch.finfo(dtype).eps / 2
    tol = u * (want.abs() + eps) + eps + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    tol[..., 2 * half:] = 0.0
    return tol


CONFIGS = [
    dict(), dict(layout="interleaved"), dict(rotary_dim=16), dict(rotary_dim=96, layout="interleaved"),
    dict(rotary_dim=48, scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
    dict(rotary_dim=64, layout="interleaved", scaling="by_parts", factor=8.0, original=4096),
    dict(rotary_dim=112, base=500000.0),
]


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rotation(lib, config, dtype):
    config = RotaryConfig(**config)
    op = Rotary(config, lib)
    torch.manual_seed(1)
    for tokens, heads, far in ((1, 1, 5), (7, 3, 1 << 20), (300, 12, 131072), (33, 5, 1 << 24)):
        say(f"case rotary {tokens} x {heads} to {far} {config} {dtype}")
        x = torch.randn(tokens, heads, 128).to(TYPES[dtype])
        positions = torch.randint(0, far, (tokens,)).int()
        for backward in (False, True):
            want = rotate64(x, positions, config.frequencies(), config.magnitude, config.layout, backward)
            got = op(x.cuda(), positions.cuda(), backward=backward)
            compare(got.cpu(), want, bound(x, want, config))
        xg = x.cuda()
        assert op(xg, positions.cuda(), out=xg) is xg
        want = rotate64(x, positions, config.frequencies(), config.magnitude, config.layout)
        compare(xg.cpu(), want, bound(x, want, config))


@pytest.mark.parametrize("layout", ["tokens", "heads"])
@pytest.mark.parametrize("tokens,heads,page,dtype", [(1, (12, 1), 16, "fp16"), (50, (8, 2), 64, "bf16"),
                                                     (700, (4, 4), 32, "fp16"), (5000, (24, 2), 256, "bf16")])
def test_append(lib, tokens, heads, page, dtype, layout):
    config = RotaryConfig(rotary_dim=64)
    say(f"case append {tokens} {heads} {page} {dtype} {layout}")
    torch.manual_seed(2)
    q, k, v = (torch.randn(tokens, h, 128).to(TYPES[dtype]) for h in (heads[0], heads[1], heads[1]))
    positions = torch.randint(0, 100000, (tokens,)).int()
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page)[:tokens].int()
    slots[::7] = -1
    slots[3::11] = pages * page + 5              # past the cache: not stored
    k_cache, v_cache = (torch.full((pages, page, heads[1], 128), 7.0, dtype=TYPES[dtype]) for _ in range(2))

    def stored(c):
        return c.transpose(1, 2).contiguous().cuda().transpose(1, 2) if layout == "heads" else c.cuda()

    kg, vg = stored(k_cache), stored(v_cache)
    # Rows of one projection: q, k and v side by side.
    qkv = torch.cat([q, k, v], 1).cuda()
    got = Rotary(config, lib).append(qkv[:, :heads[0]], qkv[:, heads[0]:heads[0] + heads[1]],
                                     qkv[:, heads[0] + heads[1]:], positions.cuda(), slots.cuda(), kg, vg)

    def turned(x):
        return rotate64(x, positions, config.frequencies(), 1.0, config.layout)

    compare(got.cpu(), turned(q), bound(q, turned(q), config))
    kept = [t for t in range(tokens) if 0 <= slots[t] < pages * page]
    want_k, want_v = k_cache.double(), v_cache.double()
    tol = torch.zeros_like(want_k)
    rows, allowed = turned(k), bound(k, turned(k), config)
    for t in kept:
        at = (int(slots[t]) // page, int(slots[t]) % page)
        want_k[at], want_v[at], tol[at] = rows[t], v[t].double(), allowed[t]
    compare(kg.cpu(), want_k, tol)
    assert torch.equal(vg.cpu().double(), want_v)
