"""A paged K/V cache and the attention over it: the serving operators of
``fa_amd.serving`` in the order a model's step runs them.

A step of every running request, prompts in pieces and single tokens alike::

    cache = PagedCache(CacheConfig(layers=2, heads_q=12, heads_kv=1, pages=4096))
    plan = cache.begin(new, tokens, max_new)      # pages and slots for the new tokens
    for layer in range(2):
        o = cache.attend(layer, q, k, v)          # [tokens, heads_q, 128]
    cache.release(request)                        # when a request has ended

Nothing waits for the GPU or copies from it: lengths, block tables and the list
of free pages live there, and a step of fixed ``tokens`` can be captured in a
graph (``begin`` included: it updates the cache's state in place).
"""

from dataclasses import dataclass, field

from fa_amd.serving import (DIM, PagedAttention, PagedConfig, PagePlanner, Rotary, RotaryConfig,
                            load_library)


@dataclass(frozen=True)
class CacheConfig:
    layers: int
    heads_q: int
    heads_kv: int
    pages: int                       # of every layer, shared by the requests
    page_size: int = 64
    max_batch: int = 64              # requests that run at once
    max_length: int = 131072         # tokens of a request, at most
    dtype: str = "float16"           # or "bfloat16"
    rotary: RotaryConfig = field(default_factory=RotaryConfig)
    attention: PagedConfig = field(default_factory=PagedConfig)

    def __post_init__(self):
        for name in ("layers", "heads_q", "heads_kv", "pages", "page_size", "max_batch", "max_length"):
            if not isinstance(getattr(self, name), int) or getattr(self, name) < 1:
                raise ValueError(f"{name} must be a positive int")
        if self.heads_q % self.heads_kv:
            raise ValueError("heads_q must be a multiple of heads_kv")
        if self.dtype not in ("float16", "bfloat16"):
            raise ValueError(f"unknown element type {self.dtype!r}")


class PagedCache:
    """The caches of all layers, the requests' block tables and lengths, and the
    operators over them. Request numbers are 0 .. max_batch - 1; one that holds no
    token is free."""

    def __init__(self, config, device="cuda", library=None):
        import torch

        lib = load_library(library)
        self.config = config
        self.planner = PagePlanner(config.page_size, lib)
        self.rotary = Rotary(config.rotary, lib)
        self.attention = PagedAttention(config.attention, lib)
        device = torch.device(device)
        shape = (config.layers, config.pages, config.page_size, config.heads_kv, DIM)
        dtype = getattr(torch, config.dtype)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        ints = dict(dtype=torch.int32, device=device)
        self.table = torch.full((config.max_batch, -(-config.max_length // config.page_size)), -1, **ints)
        self.lengths = torch.zeros(config.max_batch, **ints)
        # Free pages from index `taken` on, behind those in use.
        self.pages = torch.arange(config.pages, **ints)
        self.taken = torch.zeros(1, **ints)
        self.plan = None
        self.max_new = 1

    def begin(self, new, tokens, max_new):
        """Makes room for ``new`` [max_batch] further tokens of every request (0: it
        sits out) and returns the step's ``PagePlan``: positions and slots of
        ``tokens`` rows, request by request (more than the sum of ``new``: the
        rest belongs to none). ``max_new`` bounds the entries of ``new``. When the
        pages do not suffice, the plan's ``taken`` exceeds their number and the rows
        that read a missing one get NaN, as all rows of a request longer than
        ``max_length`` do, until release()."""
        self.plan = self.planner(self.lengths, new, self.table, self.pages, self.taken, tokens)
        self.lengths.copy_(self.plan.key_lengths)
        self.taken.copy_(self.plan.taken)
        self.max_new = max_new
        return self.plan

    def attend(self, layer, q, k, v, return_lse=False):
        """Stores the step's k and v [tokens, heads_kv, 128] of a layer, k rotated, and
        returns the attention of q [tokens, heads_q, 128], rotated, over the
        requests' tokens so far."""
        if self.plan is None:
            raise RuntimeError("begin() comes before attend()")
        plan = self.plan
        rotated = self.rotary.append(q, k, v, plan.positions, plan.slots, self.k[layer], self.v[layer])
        return self.attention(rotated, self.k[layer], self.v[layer], self.table, plan.query_starts,
                              plan.key_lengths, self.max_new, return_lse=return_lse)

    def release(self, request):
        """Ends a request: its pages are free again and its number too. The list of
        pages is made anew from the block tables, so pages that were counted as taken
        but never entered (see ``begin``) are free again as well."""
        import torch

        if not 0 <= request < self.config.max_batch:
            raise ValueError(f"request must be 0 .. {self.config.max_batch - 1}")
        self.table[request] = -1
        self.lengths[request] = 0
        # A flag a page, and one that the empty entries (-1) set.
        used = torch.zeros(self.config.pages + 1, dtype=torch.int32, device=self.table.device)
        used[self.table.flatten().long()] = 1
        used = used[:-1]
        self.pages.copy_(torch.sort(used, descending=True, stable=True).indices)
        self.taken.copy_(used.sum())
