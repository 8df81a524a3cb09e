"""The serving library on the host: it exports and binds what its header declares,
and refuses what its header refuses before anything touches a GPU; the Python
operators' own refusals; rotary frequencies; the plain page plan.

No call here gets as far as a launch."""

import ctypes as C
import math
import os
import re
from pathlib import Path

import pytest
import torch

from fa_amd import build, serving
from fa_amd.cache import CacheConfig
from fa_amd.serving import (PagedAttention, PagedConfig, PagePlanner, Rotary, RotaryConfig,
                            WindowAttention, WindowConfig)

import serving_reference

HEADER = Path(__file__).resolve().parent.parent / "include" / "fa_serve.h"
A = 4096                                     # an aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    path = os.environ.get("FA_TEST_SERVE_LIBRARY")
    if not path:
        if not build.up_to_date(build.SERVING):
            build.build(target=build.SERVING)
        path = build.SERVING.library
    return serving.load_library(path)


def test_header_declares_the_binding_signatures():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    found = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(fa_\w+)\s*\(", text, flags=re.M))
    assert found == set(serving.SIGNATURES)


def test_struct_sizes_follow_the_header():
    # int64 fields, then the 4-byte ones in pairs, then strides.
    assert C.sizeof(serving.FaPagePlan) == 6 * 8
    assert C.sizeof(serving.FaRotary) == 6 * 8 + 4 * 4 + (2 * 4 + 3 * 2) * 8
    assert C.sizeof(serving.FaPaged) == 11 * 8 + 2 * 4 + (2 * 2 + 3 * 2) * 8
    assert C.sizeof(serving.FaWindow) == 7 * 8 + 2 * 4 + 8 + 12 * 8


def test_every_status_has_a_message(lib):
    codes = re.findall(r"FA_SERVE_(?:OK|ERR_\w+) = (\d+)", HEADER.read_text())
    messages = [lib.fa_serve_strerror(int(c)) for c in codes]
    assert len(set(messages)) == len(codes) > 10 and lib.fa_serve_strerror(99) == b"unknown status"


def plan_call(lib, batch=4, tokens=10, page=16, width=8, stride=8, count=5, **over):
    prob = serving.FaPagePlan(batch, tokens, page, width, stride, count)
    args = dict(past=A, fresh=A, table=A, pages=A, taken=A, starts=A, lengths=A, positions=A, slots=A, out=A)
    args.update(over)
    return lib.fa_plan_pages(prob, *args.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), 2), (dict(batch=4097), 2), (dict(tokens=-1), 2), (dict(tokens=(1 << 30) + 1), 2),
    (dict(page=8), 4), (dict(page=48), 4), (dict(page=1 << 17), 4), (dict(width=0), 2),
    (dict(stride=7), 11), (dict(count=-1), 2), (dict(past=None), 1), (dict(slots=None), 1),
    (dict(pages=None), 1), (dict(out=None), 1), (dict(table=A + 2), 5), (dict(slots=A + 1), 5),
])
def test_plan_refusals(lib, kw, code):
    assert plan_call(lib, **kw) == code


def rotary_call(lib, tokens=3, heads_q=4, heads_kv=2, dim=64, pages=4, page=16, factor=1.0, kind=0, layout=0,
                qs=(512, 128), kc=(4096, 256, 128), **over):
    prob = serving.FaRotary(tokens, heads_q, heads_kv, dim, pages, page, factor, kind, layout, 0)
    prob.q[:], prob.q_out[:], prob.k[:], prob.v[:] = qs, (512, 128), (256, 128), (256, 128)
    prob.k_cache[:], prob.v_cache[:] = kc, (4096, 256, 128)
    args = dict(q=A, q_out=A, k=A, v=A, positions=A, slots=A, turns=A, k_cache=A, v_cache=A)
    args.update(over)
    return lib.fa_rotary_append(prob, *args.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), 2), (dict(heads_q=-1), 2), (dict(heads_q=0, heads_kv=0), 2), (dict(heads_q=4097), 2),
    (dict(dim=8), 9), (dict(dim=40), 9), (dict(dim=144), 9), (dict(layout=2), 9), (dict(kind=2), 3),
    (dict(page=17), 4), (dict(pages=-1), 2), (dict(qs=(512, 100)), 5), (dict(qs=(-512, 128)), 11),
    (dict(kc=(4096, 1 << 41, 128)), 11), (dict(q=None), 1), (dict(turns=None), 1), (dict(slots=None), 1),
    (dict(v_cache=None), 1), (dict(k=A + 8), 5), (dict(turns=A + 4), 5), (dict(positions=A + 2), 5),
])
def test_rotary_refusals(lib, kw, code):
    assert rotary_call(lib, **kw) == code


def test_no_tokens_is_no_launch(lib):
    assert rotary_call(lib, tokens=0) == 0


def paged_problem(batch=3, tokens=9, heads_q=8, heads_kv=2, max_new=4, pages=10, page=16, width=8, stride=8,
                  window=0, sinks=0, scale=0.1, kind=0, qs=(1024, 128), kc=(4096, 256, 128)):
    prob = serving.FaPaged(batch, tokens, heads_q, heads_kv, max_new, pages, page, width, stride, window,
                           sinks, scale, kind)
    prob.q[:], prob.o[:], prob.k_cache[:], prob.v_cache[:] = qs, (1024, 128), kc, (4096, 256, 128)
    return prob


def paged_call(lib, ws=A, size=None, q=A, k=A, v=A, table=A, starts=A, lengths=A, o=A, lse=A, **kw):
    prob = paged_problem(**kw)
    need = C.c_uint64()
    rc = lib.fa_paged_workspace_bytes(prob, C.byref(need))
    if rc:
        return rc
    return lib.fa_paged_fwd(prob, q, k, v, table, starts, lengths, o, lse, ws,
                            need.value if size is None else need.value + size, None)


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), 2), (dict(batch=4097), 2), (dict(heads_q=7), 2), (dict(heads_kv=0), 2), (dict(max_new=0), 2),
    (dict(tokens=1 << 30), 2), (dict(pages=-1), 2), (dict(width=0), 2), (dict(width=1 << 30), 2),
    (dict(page=24), 4), (dict(kind=3), 3), (dict(window=-1), 7), (dict(sinks=3), 7),
    (dict(window=3, sinks=-1), 7), (dict(scale=0.0), 8), (dict(scale=float("nan")), 8),
    (dict(scale=float("inf")), 8), (dict(stride=5), 11), (dict(kc=(4096, 64, 128)), 11),
    (dict(kc=(1 << 31, 256, 128)), 11), (dict(kc=(4096, 1 << 25, 128)), 11), (dict(kc=(4096, 260, 128)), 5),
    (dict(q=None), 1), (dict(table=None), 1), (dict(lengths=None), 1), (dict(o=None), 1),
    (dict(k=A + 8), 5), (dict(lse=A + 2), 5), (dict(starts=A + 1), 5), (dict(ws=None), 6), (dict(size=-1), 6),
    (dict(batch=4096, heads_q=4096, heads_kv=4096, width=1 << 24), 2),
])
def test_paged_refusals(lib, kw, code):
    assert paged_call(lib, **kw) == code


def window_call(lib, batch=2, heads_q=8, heads_kv=2, seq_q=5, seq_k=9, window=4, sinks=0, scale=0.1, kind=0,
                causal=2, ks=(2304, 1152, 128), q=A, k=A, v=A, o=A, lse=A, ws=A, size=0):
    prob = serving.FaWindow(batch, heads_q, heads_kv, seq_q, seq_k, window, sinks, scale, kind, causal)
    prob.q[:], prob.o[:], prob.k[:], prob.v[:] = (5120, 640, 128), (5120, 640, 128), ks, (2304, 1152, 128)
    need = C.c_uint64()
    rc = lib.fa_window_workspace_bytes(prob, C.byref(need))
    if rc:
        return rc
    return lib.fa_window_fwd(prob, q, k, v, o, lse, ws, need.value + size, None)


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), 2), (dict(heads_q=9), 2), (dict(seq_q=0), 2), (dict(seq_k=1 << 30), 2), (dict(window=0), 7),
    (dict(sinks=-1), 7), (dict(scale=-1.0), 8), (dict(kind=9), 3), (dict(causal=0), 12), (dict(causal=3), 12),
    (dict(ks=(2304, 1152, 64)), 11), (dict(ks=(2304, 1156, 128)), 5), (dict(q=None), 1), (dict(v=A + 4), 5),
    (dict(ws=None), 6), (dict(size=-1), 6), (dict(seq_q=1 << 27), 2),
])
def test_window_refusals(lib, kw, code):
    assert window_call(lib, **kw) == code


def test_null_problems(lib):
    size = C.c_uint64()
    assert lib.fa_paged_workspace_bytes(None, C.byref(size)) == 1
    assert lib.fa_window_workspace_bytes(None, C.byref(size)) == 1
    assert lib.fa_paged_workspace_bytes(paged_problem(), None) == 1
    assert lib.fa_plan_pages(None, *[A] * 10, None) == 1


def test_workspace_follows_what_the_call_may_launch(lib):
    def paged(**kw):
        size = C.c_uint64()
        assert lib.fa_paged_workspace_bytes(paged_problem(**kw), C.byref(size)) == 0
        return size.value

    few = paged(max_new=1)                    # the row kernel's pieces alone
    assert 0 < few < 32 << 20
    assert paged(max_new=1, batch=64, tokens=64) == few
    one = paged(batch=1, tokens=2000, max_new=2000)   # the tile kernel's parts alone
    assert 64 << 20 < one < 80 << 20
    assert paged(batch=3, tokens=2000, max_new=2000) == one + few


# The Python operators.

def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_operators_refuse_cpu_tensors(lib):
    with pytest.raises(ValueError, match="one GPU"):
        PagePlanner(16, lib)(ints(2), ints(2), ints(2, 4), ints(5), ints(1), 3)
    with pytest.raises(ValueError, match="one GPU"):
        Rotary(library=lib)(half(3, 2, 128), ints(3))
    with pytest.raises(ValueError, match="one GPU"):
        PagedAttention(library=lib)(half(3, 2, 128), half(4, 16, 1, 128), half(4, 16, 1, 128), ints(2, 4),
                                    ints(3), ints(2), 1)
    with pytest.raises(ValueError, match="one GPU"):
        WindowAttention(WindowConfig(4), lib)(half(1, 2, 3, 128), half(1, 1, 5, 128), half(1, 1, 5, 128))


@pytest.mark.parametrize("kw,match", [
    (dict(past=ints(0)), "B from 1"), (dict(past=ints(2, 2)), "B from 1"), (dict(new=ints(3)), "new"),
    (dict(new=ints(2).long()), "new"), (dict(table=ints(3, 4)), "table"), (dict(table=ints(2, 0)), "table"),
    (dict(pages=ints(4, 4)), "pages"), (dict(taken=ints(2)), "taken"), (dict(tokens=-1), "tokens"),
    (dict(tokens=2.0), "tokens"), (dict(pages=ints(8)[::2]), "contiguous"),
    (dict(table=ints(1, 4).expand(2, 4)), "overlap"),
])
def test_planner_refusals(lib, kw, match):
    args = dict(past=ints(2), new=ints(2), table=ints(2, 4), pages=ints(5), taken=ints(1), tokens=3)
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        PagePlanner(16, lib)(*args.values())


@pytest.mark.parametrize("page", [0, 8, 17, 1 << 17, 16.0])
def test_planner_page_sizes(lib, page):
    with pytest.raises(ValueError, match="power of two"):
        PagePlanner(page, lib)


@pytest.mark.parametrize("kw,match", [
    (dict(q=half(3, 128)), "q must be"), (dict(q=half(3, 3, 128), k=half(4, 16, 2, 128), v=half(4, 16, 2, 128)), "multiple"), (dict(q=half(3, 2, 64)), "128"),
    (dict(q=half(3, 2, 128).float()), "FP16 or BF16"), (dict(q=half(3, 2, 128).bfloat16()), "one type"),
    (dict(q=half(3, 2, 256)[..., ::2]), "contiguous dims"), (dict(q=half(3, 2, 136)[..., 4:132]), "aligned"),
    (dict(k=half(4, 24, 1, 128)), "caches"), (dict(v=half(4, 16, 2, 128)), "caches"),
    (dict(k=half(4, 24, 1, 128), v=half(4, 24, 1, 128)), "power of two"), (dict(table=ints(2, 0)), "table"),
    (dict(starts=ints(2)), "query_starts"), (dict(lengths=ints(3)), "key_lengths"),
    (dict(lengths=torch.zeros(2)), "key_lengths"), (dict(max_new=0), "max_new"), (dict(max_new=1.5), "max_new"),
])
def test_paged_operator_refusals(lib, kw, match):
    args = dict(q=half(3, 2, 128), k=half(4, 16, 1, 128), v=half(4, 16, 1, 128), table=ints(2, 4),
                starts=ints(3), lengths=ints(2), max_new=1)
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        PagedAttention(library=lib)(*args.values())


@pytest.mark.parametrize("kw,match", [
    (dict(q=half(2, 3, 128)), "B, H, N"), (dict(k=half(1, 2, 5, 128)), "B, H, N"),
    (dict(q=half(2, 2, 3, 128)), "geometry"), (dict(q=half(1, 0, 3, 128)), "geometry"),
    (dict(k=half(1, 1, 5, 64), v=half(1, 1, 5, 64)), "contiguous dims"),
    (dict(q=half(1, 2, 3, 128).double()), "FP16 or BF16"), (dict(q=half(1, 2, 3, 128).bfloat16()), "one type"),
])
def test_window_operator_refusals(lib, kw, match):
    args = dict(q=half(1, 2, 3, 128), k=half(1, 1, 5, 128), v=half(1, 1, 5, 128))
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        WindowAttention(WindowConfig(4), lib)(*args.values())


@pytest.mark.parametrize("make", [
    lambda: PagedConfig(window=0), lambda: PagedConfig(sinks=1), lambda: PagedConfig(window=4, sinks=-1),
    lambda: PagedConfig(window=2.5), lambda: PagedConfig(window=True), lambda: WindowConfig(None),
    lambda: WindowConfig(4, causal="none"), lambda: RotaryConfig(rotary_dim=8), lambda: RotaryConfig(rotary_dim=130),
    lambda: RotaryConfig(layout="pairs"), lambda: RotaryConfig(scaling="other"), lambda: RotaryConfig(base=1.0),
    lambda: RotaryConfig(factor=0.5), lambda: RotaryConfig(turns_low=4.0, turns_high=2.0),
    lambda: CacheConfig(1, 3, 2, 8), lambda: CacheConfig(0, 2, 2, 8), lambda: CacheConfig(1, 2, 2, 8, dtype="fp8"),
])
def test_config_refusals(make):
    with pytest.raises(ValueError):
        make()


def test_scale_refusals(lib):
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            serving._check_scale(scale)


def test_rotary_frequencies():
    plain = RotaryConfig(rotary_dim=64).frequencies()
    assert len(plain) == 32 and plain[0] == 1.0
    assert plain[31] == pytest.approx(10000.0 ** (-62 / 64), rel=1e-15)
    linear = RotaryConfig(rotary_dim=64, scaling="linear", factor=4.0).frequencies()
    assert linear == [f / 4 for f in plain]
    base = RotaryConfig(rotary_dim=64, scaling="base", factor=4.0).frequencies()
    assert base[0] == plain[0] and base[31] == pytest.approx(plain[31] / 4, rel=1e-12)
    config = RotaryConfig(rotary_dim=64, scaling="by_parts", factor=4.0, original=4096)
    parts = config.frequencies()
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, p, n in zip(plain, parts, turns):
        if n >= 32:
            assert p == f
        elif n <= 1:
            assert p == pytest.approx(f / 4, rel=1e-15)
        else:
            assert f / 4 < p < f
    assert config.magnitude == pytest.approx(0.1 * math.log(4.0) + 1.0)
    assert RotaryConfig().magnitude == 1.0


def test_plain_rotation_backward_is_the_transpose():
    torch.manual_seed(0)
    config = RotaryConfig(rotary_dim=32, layout="interleaved", scaling="by_parts", factor=4.0)
    x, g = torch.randn(5, 2, 128), torch.randn(5, 2, 128)
    positions = torch.randint(0, 9999, (5,))
    args = (positions, config.frequencies(), config.magnitude, config.layout)
    y = serving_reference.rotate64(x, *args)
    gx = serving_reference.rotate64(g, *args, backward=True)
    assert (y * g).sum().item() == pytest.approx((gx * x).sum().item(), rel=1e-10)


def test_host_sanitizer_build_leaves_device_code_alone():
    flags = build.SERVING_HOSTSAN.flags
    sanitizers = [i for i, f in enumerate(flags) if f.startswith("-fsanitize")]
    assert sanitizers and all(flags[i - 1] == "-Xarch_host" for i in sanitizers)
    assert build.SERVING_HOSTSAN not in build.TARGETS and build.SERVING in build.TARGETS


def test_measured_work_counts_what_is_visible():
    from fa_amd.measure import serving as measure

    for window, sinks in ((None, 0), (1, 0), (5, 0), (5, 3), (40, 7)):
        for past, new in ((0, 1), (0, 9), (13, 4), (50, 20)):
            rows = [[j for j in range(p + 1) if window is None or j > p - window or j < sinks]
                    for p in range(past, past + new)]
            assert measure.visible_pairs(past, new, window, sinks) == sum(map(len, rows))
            keys = set().union(*rows)
            step = measure.Step("x", 4, 2, ((past, new), (3, 1)), window, sinks)
            other = [j for j in range(4) if window is None or j > 3 - window or j < sinks]
            assert measure.work(step) == (512 * ((new + 1) * 4 + 2 * (len(keys) + len(other))),
                                          512 * 4 * (sum(map(len, rows)) + len(other)))
    lines = measure.render([{"name": "x", "plan": 1.0, "store": 2.0, "attend": 3.0, "tbs": 4.0, "tflops": 5.0}],
                           "float16", "python -m fa_amd.measure.serving")
    assert lines[1] == "command: python -m fa_amd.measure.serving" and "4.00" in lines[3]


def test_refusals_of_launches_past_32_bits(lib):
    # Threads of a launch: 8 a token (rotary), 512 a tile and die (attention).
    assert rotary_call(lib, tokens=(1 << 28) + 1) == 2
    many = dict(batch=4096, heads_q=1023, heads_kv=1023, tokens=4096 * 100)
    assert paged_call(lib, **many, max_new=100, qs=(1024 * 128, 128)) == 2
    assert window_call(lib, batch=65535, heads_q=1023, heads_kv=1023, seq_q=100) == 2


@pytest.mark.parametrize("scale", [torch.tensor(0.1), "0.1", [0.1]])
def test_scale_must_be_a_number(scale):
    # A tensor would be kept by its identity, and read once.
    with pytest.raises(ValueError, match="number"):
        serving._check_scale(scale)


def small_cache(**kw):
    from fa_amd.cache import CacheConfig, PagedCache

    config = dict(layers=1, heads_q=1, heads_kv=1, pages=10, page_size=16, max_batch=3, max_length=96)
    return PagedCache(CacheConfig(**{**config, **kw}), device="cpu")


def fill(cache, new):
    """What begin() leaves in the cache's state, without the GPU."""
    plan = serving_reference.plan(cache.lengths.tolist(), new, cache.table.tolist(), cache.pages.tolist(),
                                  int(cache.taken), sum(new), cache.config.page_size)
    for name, values in (("table", plan[0]), ("lengths", plan[2]), ("taken", [plan[5]])):
        getattr(cache, name).copy_(torch.tensor(values, dtype=torch.int32))


def free_pages(cache):
    return sorted(cache.pages.tolist()[int(cache.taken):])


@pytest.mark.parametrize("steps,end", [
    ([[40, 20, 90]], 2),                      # 3 + 2 + 6 pages of 10: one is missing
    ([[90, 0, 0], [0, 50, 90]], 0),           # the missing ones belong to others
    ([[200, 16, 0]], 0),                      # longer than its table row
    ([[16, 200, 0], [16, 0, 16]], 1),
])
def test_release_after_too_much_was_asked(steps, end):
    cache = small_cache()
    for new in steps:
        fill(cache, new)
    cache.release(end)
    held = [i for row in cache.table.tolist() for i in row if i >= 0]
    assert cache.table[end].eq(-1).all() and int(cache.lengths[end]) == 0
    assert len(set(held)) == len(held)
    # Every page that no table names is free, once.
    assert free_pages(cache) == sorted(set(range(10)) - set(held))
    for request in range(3):
        cache.release(request)
    assert free_pages(cache) == list(range(10))
