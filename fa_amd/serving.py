"""Serving operators over ``libfa_serve.so``: what a program needs around the
attention forward when its keys lie in the pages of a cache.

  * ``PagePlanner``      block tables and slot maps, built on the GPU from the
                         requests' lengths;
  * ``Rotary``           rotary positions, in place of or on the way into a paged cache;
  * ``PagedAttention``   attention of every request's new tokens over its pages;
  * ``WindowAttention``  attention with a sliding window and sinks on
                         contiguous [B, H, N, 128] tensors.

They follow ``fa_amd.binding.Operator``: errors of geometry, type, device and
layout raise ``ValueError`` before any launch, a nonzero library status raises
``RuntimeError``, a call is enqueued on the current torch stream of its tensors'
device, and without the built library construction fails. Unlike it, every call
returns tensors of its own (or fills ``out``) and takes its workspace from
torch's allocator, on the call's stream, so one object may be used on several
streams and in several captured graphs at once.

FP16 and BF16, 128 dims per head. Integers are int32 tensors on the GPU: no
call waits for the GPU or copies from it. The reference has no counterpart.
"""

import ctypes as C
import math
import numbers
from collections import namedtuple
from dataclasses import dataclass

from fa_amd.binding import SIGNATURES_KEPT

DIM = 128
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "base", "by_parts")
CAUSAL = {"top_left": 1, "bottom_right": 2}


class FaPagePlan(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("batch", "tokens", "page_size", "max_pages",
                                         "table_stride", "pages_count")]


class FaRotary(C.Structure):
    _fields_ = [("tokens", C.c_int64), ("heads_q", C.c_int64), ("heads_kv", C.c_int64),
                ("rotary_dim", C.c_int64), ("pages", C.c_int64), ("page_size", C.c_int64),
                ("factor", C.c_float), ("type", C.c_int32), ("layout", C.c_int32),
                ("backward", C.c_int32), ("q", C.c_int64 * 2), ("q_out", C.c_int64 * 2),
                ("k", C.c_int64 * 2), ("v", C.c_int64 * 2), ("k_cache", C.c_int64 * 3),
                ("v_cache", C.c_int64 * 3)]


class FaPaged(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("batch", "tokens", "heads_q", "heads_kv", "max_new",
                                         "pages", "page_size", "max_pages", "table_stride",
                                         "window", "sinks")] + \
               [("scale", C.c_float), ("type", C.c_int32), ("q", C.c_int64 * 2),
                ("o", C.c_int64 * 2), ("k_cache", C.c_int64 * 3), ("v_cache", C.c_int64 * 3)]


class FaWindow(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("batch", "heads_q", "heads_kv", "seq_q", "seq_k",
                                         "window", "sinks")] + \
               [("scale", C.c_float), ("type", C.c_int32), ("causal", C.c_int32),
                ("q", C.c_int64 * 3), ("k", C.c_int64 * 3), ("v", C.c_int64 * 3),
                ("o", C.c_int64 * 3)]


P = C.c_void_p
# Every symbol include/fa_serve.h declares, with its ctypes signature.
SIGNATURES = {
    "fa_plan_pages": (C.c_int, [C.POINTER(FaPagePlan)] + [P] * 11),
    "fa_rotary_append": (C.c_int, [C.POINTER(FaRotary)] + [P] * 10),
    "fa_paged_workspace_bytes": (C.c_int, [C.POINTER(FaPaged), C.POINTER(C.c_uint64)]),
    "fa_paged_fwd": (C.c_int, [C.POINTER(FaPaged)] + [P] * 9 + [C.c_uint64, P]),
    "fa_window_workspace_bytes": (C.c_int, [C.POINTER(FaWindow), C.POINTER(C.c_uint64)]),
    "fa_window_fwd": (C.c_int, [C.POINTER(FaWindow)] + [P] * 6 + [C.c_uint64, P]),
    "fa_serve_strerror": (C.c_char_p, [C.c_int]),
}

PagePlan = namedtuple("PagePlan", "query_starts key_lengths positions slots taken")


def load_library(path=None):
    """The serving library at `path` (default: the built one) with its signatures."""
    if path is None:
        from fa_amd import build

        path = build.SERVING.library
        if not path.is_file():
            raise FileNotFoundError(f"{path} is not built (python -m fa_amd.build)")
    lib = C.CDLL(str(path), mode=C.RTLD_LOCAL)
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    return lib


def _type(tensor):
    import torch

    if tensor.dtype == torch.float16:
        return 0
    if tensor.dtype == torch.bfloat16:
        return 1
    raise ValueError("tensors must be FP16 or BF16")


def _on_gpu(device, *tensors):
    if device.type != "cuda" or any(t.device != device for t in tensors):
        raise ValueError("all tensors must be on one GPU")


def _ints(shapes, **tensors):
    """int32 and contiguous in the last dimension, of the given shape (None: any size)."""
    import torch

    for name, t in tensors.items():
        want = shapes[name]
        if t.dtype != torch.int32 or t.ndim != len(want) or \
                any(w is not None and n != w for n, w in zip(t.shape, want)):
            dims = ", ".join("*" if w is None else str(w) for w in want)
            raise ValueError(f"{name} must be an int32 tensor [{dims}]")
        if t.numel() and t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{name} must be contiguous")


def _strides(tensor, name):
    """Strides in front of the 128 contiguous dims."""
    st = tensor.stride()
    if tensor.shape[-1] != DIM or (tensor.numel() and (
            st[-1] != 1 or any(s % 8 or s < 0 for s in st[:-1]) or tensor.data_ptr() % 16)):
        raise ValueError(f"{name} must have {DIM} contiguous dims and 16-byte aligned rows")
    return tuple(min(s, 1 << 40) for s in st[:-1])


def _signature(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


class _Operator:
    """What the operators share: the library, what a call derives from its
    signature (kept for the last ``SIGNATURES_KEPT`` of them) and the launch."""

    def __init__(self, library):
        self.lib = library if isinstance(library, C.CDLL) else load_library(library)
        self.plans = {}
        self.streams = {}        # (device index, raw stream) -> torch stream

    def check(self, status, where):
        if status:
            raise RuntimeError(f"{where}: {status} ({self.lib.fa_serve_strerror(status).decode()})")

    def keep(self, key, plan):
        if len(self.plans) >= SIGNATURES_KEPT:
            self.plans.clear()
        self.plans[key] = plan
        return plan

    def launch(self, fn, args, device, tensors):
        """fn(*args, stream) with `device` current. The tensors, which may come from
        other streams, are kept from being reused before it has run."""
        import torch

        index = device.index
        if index != torch.cuda.current_device():
            with torch.cuda.device(index):
                return self.launch(fn, args, device, tensors)
        raw = torch._C._cuda_getCurrentRawStream(index)
        stream = self.streams.get((index, raw))
        if stream is None:
            if len(self.streams) >= 64:
                self.streams.clear()
            stream = self.streams[index, raw] = torch.cuda.current_stream(index)
        status = fn(*args, raw)
        if status:
            self.check(status, fn.__name__)
        for t in tensors:
            t.record_stream(stream)


ALIGN_ERROR = f"rows of {DIM} dims must be 16-byte aligned"
OUT_ERROR = "out must not be a tensor that the call reads"


class PagePlanner(_Operator):
    """Callable ``(past, new, table, pages, taken, tokens) -> PagePlan``: pages
    and slots for the requests' new tokens (``fa_plan_pages``).

    past, new    [B] tokens a request holds and gets
    table        [B, max_pages] block table; the new pages are entered in place
    pages        free pages, given out in order from index ``taken`` [1] on
    tokens       length of the positions and slots to make (at least the sum
                 of ``new``; the rest get position 0 and slot -1)

    The plan has ``query_starts`` [B + 1], ``key_lengths`` [B], ``positions``
    and ``slots`` [tokens] and ``taken`` [1], the next call's. ``taken`` beyond
    ``len(pages)`` means that the pages did not suffice: the entries and
    slots past the last one are -1, and attention over them gives NaN.
    ``page_size`` is a power of two from 16 to 65536, B at most 4096."""

    MAX_BATCH = 4096

    def __init__(self, page_size, library=None):
        super().__init__(library)
        if not isinstance(page_size, int) or not 16 <= page_size <= 65536 or \
                page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 65536")
        self.page_size = page_size

    def __call__(self, past, new, table, pages, taken, tokens):
        import torch

        # One lookup stands for the checks of a signature met before.
        key = (past.shape, past.stride(), past.dtype, past.device, new.shape, new.stride(),
               new.dtype, new.device, table.shape, table.stride(), table.dtype, table.device,
               pages.shape, pages.stride(), pages.dtype, pages.device, taken.shape, taken.stride(),
               taken.dtype, taken.device, tokens)
        plan = self.plans.get(key)
        if plan is None:
            plan = self.keep(key, self.plan(past, new, table, pages, taken, tokens))
        prob, sizes, total = plan
        device = past.device
        made = torch.empty(total, dtype=torch.int32, device=device)
        at = made.data_ptr()
        lengths = at + 4 * sizes[0]
        positions = lengths + 4 * sizes[1]
        self.launch(self.lib.fa_plan_pages,
                    (prob, past.data_ptr(), new.data_ptr(), table.data_ptr(), pages.data_ptr(),
                     taken.data_ptr(), at, lengths, positions, positions + 4 * tokens,
                     at + 4 * (total - 1)), device, (past, new, table, pages, taken))
        return PagePlan(*made.split_with_sizes(sizes))

    def plan(self, past, new, table, pages, taken, tokens):
        if past.ndim != 1 or not 1 <= past.shape[0] <= self.MAX_BATCH:
            raise ValueError(f"past must be [B] with B from 1 to {self.MAX_BATCH}")
        batch = past.shape[0]
        _ints({"past": (batch,), "new": (batch,), "table": (batch, None), "pages": (None,),
               "taken": (1,)}, past=past, new=new, table=table, pages=pages, taken=taken)
        if table.shape[1] < 1 or (batch > 1 and table.stride(0) < table.shape[1]):
            raise ValueError("table must have rows of one page or more that do not overlap")
        if not isinstance(tokens, int) or not 0 <= tokens <= 1 << 30:
            raise ValueError("tokens must be an int from 0 to 2^30")
        _on_gpu(past.device, new, table, pages, taken)
        # One allocation: starts, lengths, positions, slots, taken.
        sizes = [batch + 1, batch, tokens, tokens, 1]
        return FaPagePlan(batch, tokens, self.page_size, table.shape[1],
                          max(table.stride(0), table.shape[1]), pages.shape[0]), sizes, sum(sizes)


@dataclass(frozen=True)
class RotaryConfig:
    """``rotary_dim`` dims of every head are rotated (a multiple of 16 up to 128),
    in pairs (i, i + rotary_dim / 2), ``layout`` "half", or (2i, 2i + 1),
    "interleaved"; pair i turns by ``base ** (-2 i / rotary_dim)`` radians a
    position. For contexts ``factor`` times longer than the ``original`` one,
    ``scaling``:

      "linear"    positions divided by ``factor``;
      "base"      ``base`` raised by ``factor ** (rotary_dim / (rotary_dim - 2))``,
                  which divides the slowest pair's turns by ``factor`` and
                  leaves the fastest pair alone;
      "by_parts"  pairs that turn fewer than ``turns_low`` times over the
                  original context divided by ``factor``, those that turn
                  more than ``turns_high`` times left alone, in between in
                  proportion to i; rotated values times 0.1 ln(factor) + 1."""
    rotary_dim: int = DIM
    base: float = 10000.0
    layout: str = "half"
    scaling: str = "none"
    factor: float = 1.0
    original: int = 4096
    turns_low: float = 1.0
    turns_high: float = 32.0

    def __post_init__(self):
        if not isinstance(self.rotary_dim, int) or self.rotary_dim % 16 or \
                not 16 <= self.rotary_dim <= DIM:
            raise ValueError(f"rotary_dim must be a multiple of 16 from 16 to {DIM}")
        if self.layout not in LAYOUTS:
            raise ValueError(f"unknown rotary layout {self.layout!r}")
        if self.scaling not in SCALINGS:
            raise ValueError(f"unknown scaling {self.scaling!r}")
        if not (self.base > 1 and math.isfinite(self.base)):
            raise ValueError("base must be finite and above 1")
        if not (self.factor >= 1 and math.isfinite(self.factor)):
            raise ValueError("factor must be finite and at least 1")
        if not 0 < self.turns_low < self.turns_high or self.original < 1:
            raise ValueError("turns_low must be positive and below turns_high, original positive")

    def frequencies(self):
        """Radians a position of every pair, as Python floats (64 bits)."""
        half = self.rotary_dim // 2
        base = self.base
        if self.scaling == "base":
            base *= self.factor ** (self.rotary_dim / (self.rotary_dim - 2))
        freq = [base ** (-i / half) for i in range(half)]
        if self.scaling == "linear":
            return [f / self.factor for f in freq]
        if self.scaling == "by_parts":
            # The (fractional) pair that turns n times over the original context.
            def pair(n):
                return half * math.log(self.original / (2 * math.pi * n)) / math.log(base)

            low, high = pair(self.turns_high), pair(self.turns_low)
            out = []
            for i, f in enumerate(freq):
                ramp = min(1.0, max(0.0, (i - low) / (high - low)))
                out.append(f / self.factor * ramp + f * (1.0 - ramp))
            return out
        return freq

    @property
    def magnitude(self):
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "by_parts" else 1.0


class Rotary(_Operator):
    """Rotary positions of ``config`` (``fa_rotary_append``).

    ``rotary(x, positions)`` rotates x [T, H, 128] (any strides of T and H) at
    ``positions`` [T]; with ``backward=True`` it is the rotation's transpose,
    which takes a gradient of the rotated tensor to one of x. ``out`` may be x
    (with its strides), and overlaps x in no other way.

    ``rotary.append(q, k, v, positions, slots, k_cache, v_cache)`` returns q
    rotated and stores k, rotated, and v at ``slots`` [T] of the caches
    [pages, page_size, heads, 128] (any strides); tokens with a slot that is
    negative or past the cache are not stored. Slots of one call that are stored
    must be distinct."""

    def __init__(self, config=RotaryConfig(), library=None):
        super().__init__(library)
        self.config = config
        self.turns = {}          # device -> FP64 turns a position of every pair

    def turns_on(self, device):
        import torch

        turns = self.turns.get(device)
        if turns is None:
            values = [f / (2 * math.pi) for f in self.config.frequencies()]
            turns = torch.tensor(values, dtype=torch.float64).to(device)
            # Other streams may use it from here on.
            torch.cuda.current_stream(device).synchronize()
            self.turns[device] = turns
        return turns

    def __call__(self, x, positions, backward=False, out=None):
        import torch

        key = (x.shape, x.stride(), x.dtype, x.device, _signature(positions), backward,
               _signature(out))
        plan = self.plans.get(key)
        if plan is None:
            plan = self.keep(key, self.plan(x, positions, out, backward))
        prob, turns = plan
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        xp, op = x.data_ptr(), out.data_ptr()
        if (xp | op) % 16:
            raise ValueError(ALIGN_ERROR)
        self.launch(self.lib.fa_rotary_append,
                    (prob, xp, op, None, None, positions.data_ptr(), None, turns.data_ptr(), None,
                     None), x.device, (x, out, positions))
        return out

    def append(self, q, k, v, positions, slots, k_cache, v_cache, out=None):
        import torch

        key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device,
               v.shape, v.stride(), v.dtype, v.device, positions.shape, positions.stride(),
               positions.dtype, positions.device, slots.shape, slots.stride(), slots.dtype,
               slots.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
               v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device, _signature(out))
        plan = self.plans.get(key)
        if plan is None:
            plan = self.keep(key, self.plan_append(q, k, v, positions, slots, k_cache, v_cache, out))
        prob, turns = plan
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        qp, op, kp, vp = q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr()
        kc, vc = k_cache.data_ptr(), v_cache.data_ptr()
        if (qp | op | kp | vp | kc | vc) % 16:
            raise ValueError(ALIGN_ERROR)
        self.launch(self.lib.fa_rotary_append,
                    (prob, qp, op, kp, vp, positions.data_ptr(), slots.data_ptr(), turns.data_ptr(),
                     kc, vc), q.device, (q, k, v, out, positions, slots, k_cache, v_cache))
        return out

    def plan(self, x, positions, out, backward=False):
        if x.ndim != 3 or not 1 <= x.shape[1] <= 4096:
            raise ValueError(f"x must be [T, H, {DIM}]")
        tokens, heads, _ = x.shape
        kind, strides = _type(x), _strides(x, "x")
        _ints({"positions": (tokens,)}, positions=positions)
        _on_gpu(x.device, positions)
        if out is None:
            out_strides = (heads * DIM, DIM)
        else:
            if out.shape != x.shape or out.dtype != x.dtype:
                raise ValueError("out must have the shape and type of what is rotated")
            _on_gpu(x.device, out)
            out_strides = _strides(out, "out")
            if any(s < DIM for s, n in zip(out_strides, out.shape) if n > 1):
                raise ValueError("out must not overlap itself")
        prob = FaRotary(tokens=tokens, heads_q=heads, rotary_dim=self.config.rotary_dim,
                        factor=self.config.magnitude, type=kind,
                        layout=LAYOUTS[self.config.layout], backward=bool(backward))
        prob.q[:], prob.q_out[:] = strides, out_strides
        return prob, self.turns_on(x.device)

    def plan_append(self, q, k, v, positions, slots, k_cache, v_cache, out):
        prob, turns = self.plan(q, positions, out)
        tokens = q.shape[0]
        if k.ndim != 3 or k.shape != v.shape or k.shape[0] != tokens or not 1 <= k.shape[1] <= 4096:
            raise ValueError(f"k and v must be [T, heads, {DIM}] with q's T")
        _check_caches(k_cache, v_cache, k.shape[1])
        if not q.dtype == k.dtype == v.dtype == k_cache.dtype == v_cache.dtype:
            raise ValueError("q, k, v and the caches must have one type")
        _ints({"slots": (tokens,)}, slots=slots)
        strides = [_strides(t, n) for t, n in ((k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache"))]
        _on_gpu(q.device, k, v, slots, k_cache, v_cache)
        prob.heads_kv, prob.pages, prob.page_size = k.shape[1], k_cache.shape[0], k_cache.shape[1]
        prob.k[:], prob.v[:], prob.k_cache[:], prob.v_cache[:] = strides
        return prob, turns


def _check_caches(k_cache, v_cache, heads):
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.shape[2] != heads:
        raise ValueError(f"caches must be [pages, page_size, {heads}, {DIM}]")
    size = k_cache.shape[1]
    if not 16 <= size <= 65536 or size & (size - 1):
        raise ValueError("page_size must be a power of two from 16 to 65536")


def _check_mask(window, sinks):
    for name, value in (("window", window), ("sinks", sinks)):
        if value is not None and (not isinstance(value, int) or isinstance(value, bool)):
            raise ValueError(f"{name} must be an int")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1")
    if sinks < 0 or (sinks and window is None):
        raise ValueError("sinks must not be negative, and need a window")


def _check_scale(scale):
    if scale is not None and not isinstance(scale, numbers.Real):
        raise ValueError("scale must be a number")
    scale = DIM ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be finite and positive")
    return scale


@dataclass(frozen=True)
class PagedConfig:
    """A row at position p sees the keys j <= p; with a ``window``, those with
    j > p - window or j < ``sinks``."""
    window: "int | None" = None
    sinks: int = 0

    def __post_init__(self):
        _check_mask(self.window, self.sinks)


class PagedAttention(_Operator):
    """Callable ``(q, k_cache, v_cache, table, query_starts, key_lengths, max_new)
    -> o``: attention of every request's new tokens over its pages, which hold
    them already (``fa_paged_fwd``).

    q             [T, heads_q, 128], the requests' new rows one after another
    k_cache,      [pages, page_size, heads_kv, 128], any strides of the first
    v_cache       three dims
    table         [B, max_pages] pages of every request's tokens, in order
    query_starts  [B + 1] first row of every request, and the end
    key_lengths   [B] tokens of every request, the new ones included
    max_new       most new tokens of a request, as far as the caller knows; it
                  chooses kernels, a larger request is still computed

    Returns o [T, heads_q, 128], with ``return_lse`` also the rows'
    log-sum-exp [T, heads_q] FP32. Rows behind the last request are left as
    they were in ``out`` (undefined without ``out``; ``out`` must not overlap what
    the call reads). A row that sees no key
    gets 0 and -inf. A request that is longer than its table row, or whose table
    names a page that the cache does not have, gets NaN where that is read."""

    MAX_BATCH = 4096

    def __init__(self, config=PagedConfig(), library=None):
        super().__init__(library)
        self.config = config

    def __call__(self, q, k_cache, v_cache, table, query_starts, key_lengths, max_new, scale=None,
                 return_lse=False, out=None):
        import torch

        key = (q.shape, q.stride(), q.dtype, q.device, k_cache.shape, k_cache.stride(),
               k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype,
               v_cache.device, table.shape, table.stride(), table.dtype, table.device,
               query_starts.shape, query_starts.stride(), query_starts.dtype, query_starts.device,
               key_lengths.shape, key_lengths.stride(), key_lengths.dtype, key_lengths.device,
               max_new, scale, _signature(out))
        plan = self.plans.get(key)
        if plan is None:
            plan = self.keep(key, self.plan(q, k_cache, v_cache, table, query_starts, key_lengths,
                                            max_new, scale, out))
        prob, size = plan
        device = q.device
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=device) if return_lse else None
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        qp, kc, vc, op = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
        if (qp | kc | vc | op) % 16:
            raise ValueError(ALIGN_ERROR)
        if op and op in (qp, kc, vc):
            raise ValueError(OUT_ERROR)
        self.launch(self.lib.fa_paged_fwd,
                    (prob, qp, kc, vc, table.data_ptr(), query_starts.data_ptr(),
                     key_lengths.data_ptr(), op, lse.data_ptr() if return_lse else None,
                     ws.data_ptr(), size), device,
                    (q, k_cache, v_cache, table, query_starts, key_lengths, out))
        return (out, lse) if return_lse else out

    def plan(self, q, k_cache, v_cache, table, query_starts, key_lengths, max_new, scale, out):
        if q.ndim != 3 or q.shape[1] < 1 or k_cache.ndim != 4 or k_cache.shape[2] < 1 or \
                q.shape[1] % k_cache.shape[2] or q.shape[1] > 4096:
            raise ValueError(f"q must be [T, heads_q, {DIM}], with a multiple of the caches' heads")
        _check_caches(k_cache, v_cache, k_cache.shape[2])
        if table.ndim != 2 or not 1 <= table.shape[0] <= self.MAX_BATCH or table.shape[1] < 1:
            raise ValueError(f"table must be [B, max_pages] with B from 1 to {self.MAX_BATCH}")
        batch = table.shape[0]
        _ints({"table": (batch, None), "query_starts": (batch + 1,), "key_lengths": (batch,)},
              table=table, query_starts=query_starts, key_lengths=key_lengths)
        if batch > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("rows of table must not overlap")
        if not isinstance(max_new, int) or max_new < 1:
            raise ValueError("max_new must be a positive int")
        kind = _type(q)
        if not q.dtype == k_cache.dtype == v_cache.dtype:
            raise ValueError("q and the caches must have one type")
        strides = [_strides(t, n) for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"))]
        _on_gpu(q.device, k_cache, v_cache, table, query_starts, key_lengths)
        prob = FaPaged(batch, q.shape[0], q.shape[1], k_cache.shape[2], min(max_new, 1 << 40),
                       k_cache.shape[0], k_cache.shape[1], table.shape[1],
                       max(table.stride(0), table.shape[1]), self.config.window or 0,
                       self.config.sinks, _check_scale(scale), kind)
        prob.q[:], prob.k_cache[:], prob.v_cache[:] = strides
        prob.o[:] = _out_strides(q, out)
        size = C.c_uint64()
        self.check(self.lib.fa_paged_workspace_bytes(prob, C.byref(size)), "fa_paged_workspace_bytes")
        return prob, max(size.value, 16)


def _out_strides(q, out):
    if out is None:
        strides, n = [], DIM
        for size in reversed(q.shape[:-1]):
            strides.insert(0, n)
            n *= size
        return strides
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and type")
    _on_gpu(q.device, out)
    strides = _strides(out, "out")
    if any(s < DIM for s, n in zip(strides, out.shape) if n > 1):
        raise ValueError("out must not overlap itself")
    return strides


@dataclass(frozen=True)
class WindowConfig:
    """A row at position p sees the keys j <= p with j > p - ``window`` or
    j < ``sinks``; row i stands at p = i + Nk - Nq (``causal`` "bottom_right": the
    last row at the last key) or p = i ("top_left")."""
    window: int
    sinks: int = 0
    causal: str = "bottom_right"

    def __post_init__(self):
        _check_mask(self.window, self.sinks)
        if self.window is None:
            raise ValueError("window must be an int")
        if self.causal not in CAUSAL:
            raise ValueError(f"unknown causal mode {self.causal!r}")


class WindowAttention(_Operator):
    """Callable ``(q, k, v) -> o`` (``fa_window_fwd``): q [B, Hq, Nq, 128], k and v
    [B, Hkv, Nk, 128], any strides of the first three dims; with ``return_lse``
    also the rows' log-sum-exp [B, Hq, Nq] FP32. A row that sees no key gets 0
    and -inf. ``out`` must not overlap what the call reads."""

    def __init__(self, config, library=None):
        super().__init__(library)
        self.config = config

    def __call__(self, q, k, v, scale=None, return_lse=False, out=None):
        import torch

        key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device,
               v.shape, v.stride(), v.dtype, v.device, scale, _signature(out))
        plan = self.plans.get(key)
        if plan is None:
            plan = self.keep(key, self.plan(q, k, v, scale, out))
        prob, size = plan
        device = q.device
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=device) if return_lse else None
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        if (qp | kp | vp | op) % 16:
            raise ValueError(ALIGN_ERROR)
        if op in (qp, kp, vp):
            raise ValueError(OUT_ERROR)
        self.launch(self.lib.fa_window_fwd,
                    (prob, qp, kp, vp, op, lse.data_ptr() if return_lse else None, ws.data_ptr(),
                     size), device, (q, k, v, out))
        return (out, lse) if return_lse else out

    def plan(self, q, k, v, scale, out):
        if q.ndim != 4 or k.ndim != 4 or k.shape != v.shape:
            raise ValueError(f"q, k and v must be [B, H, N, {DIM}]")
        if min(q.shape) < 1 or min(k.shape) < 1 or k.shape[0] != q.shape[0] or \
                q.shape[1] % k.shape[1] or q.shape[1] > 4096:
            raise ValueError("invalid attention geometry")
        kind = _type(q)
        if not q.dtype == k.dtype == v.dtype:
            raise ValueError("q, k and v must have one type")
        strides = [_strides(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v"))]
        _on_gpu(q.device, k, v)
        prob = FaWindow(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2],
                        self.config.window, self.config.sinks, _check_scale(scale), kind,
                        CAUSAL[self.config.causal])
        prob.q[:], prob.k[:], prob.v[:] = strides
        prob.o[:] = _out_strides(q, out)
        size = C.c_uint64()
        self.check(self.lib.fa_window_workspace_bytes(prob, C.byref(size)), "fa_window_workspace_bytes")
        return prob, max(size.value, 16)
