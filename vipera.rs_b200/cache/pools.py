"""Device memory of the cache and its grouping.

Layers whose mixers ask for the same kind of paged memory (KV head count, head size,
window) form a group.  A group has pages of its own: one page number addresses the same
page in every layer of the group, as one block addresses every layer in the reference
(crates/vipera-backend-cpu/src/model.rs:63-70, crates/vipera-runtime/src/pipeline.rs:128-129).
Inside a group the memory is [slot in group][k or v][page][position in page][kv head][d],
the reference's layer-major order lifted to the pool (model.rs:1451-1469), so that each
layer's keys are one dense [pages * page_size, kv_heads * d] matrix.

Mixers that keep a fixed-size state get one tensor [state slots, *shape] per cache slot.
The bookkeeping (which request holds which page and which state slot) is the native
``CacheManager``; this module owns only the memory.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional, Tuple

import torch

from ..build import runtime_module
from ..errors import InvalidArgumentError, UnsupportedError
from ..kernels.ops import Q4_GROUP, Q4Pages
from ..parts.base import FixedState, PagedKV, PagedKVView, PagedQ4View, StateView, bundle_views, flatten_cache_requests


KV_TYPES = ("q4",)    # kinds of pages beside those of the run's type (None)
_Q4_ALIGN = 256       # bytes: where codes, scales and guards of 4-bit pools begin
GUARD_WORD = 0x5A5A   # fits 16 bits: the guard regions are viewed as integers of the element's width


@dataclass
class CacheGroup:
    num_kv_heads: int
    head_dim: int
    window: Optional[int]
    value_dim: int = 0       # 0: values are as long as keys
    keep_first: int = 0
    slots: List[int] = field(default_factory=list)  # cache slots (of the schedule) in this group

    @property
    def v_dim(self) -> int:
        return self.value_dim or self.head_dim

    def bytes_per_token(self, element_bytes: int, kv_type: Optional[str] = None) -> int:
        values = len(self.slots) * self.num_kv_heads * (self.head_dim + self.v_dim)
        if kv_type == "q4":
            return values // 2 + values // Q4_GROUP * 2     # a code for each value, a bfloat16 scale for each group
        return values * element_bytes


def plan_groups(cache_requests: Dict[int, object]) -> Tuple[List[CacheGroup], Dict[int, FixedState]]:
    """Sort the cache slots of a model into paged groups and fixed-state slots.  A slot that keeps
    several things (a ``CacheBundle``) appears once per member, under the key (slot, name)."""
    groups: Dict[tuple, CacheGroup] = {}
    states: Dict[object, FixedState] = {}
    flat = flatten_cache_requests(cache_requests)
    for slot, request in flat.items():
        if isinstance(request, PagedKV):
            value_dim = request.value_dim if request.value_dim and request.value_dim != request.head_dim else 0
            keep_first = int(request.keep_first or 0) if request.window else 0
            key = (request.num_kv_heads, request.head_dim, request.window, value_dim, keep_first)
            if key not in groups:
                groups[key] = CacheGroup(*key)
            groups[key].slots.append(slot)
        elif isinstance(request, FixedState):
            states[slot] = request
        else:
            raise InvalidArgumentError(f"cache slot {slot}: unknown kind of cache request {request!r}")
    return list(groups.values()), states


def check_kv_type(kv_type: Optional[str], cache_requests: Dict[int, object]) -> Optional[str]:
    """None (pages of the run's type) or "q4" (pages of 4 bits), the latter where every mixer that keeps pages takes them."""
    if kv_type is None:
        return None
    if kv_type not in KV_TYPES:
        raise InvalidArgumentError(f"the cache's type is the run's or one of {', '.join(KV_TYPES)}, not {kv_type!r}")
    paged = [(slot, r) for slot, r in flatten_cache_requests(cache_requests).items() if isinstance(r, PagedKV)]
    if not paged:
        raise UnsupportedError("no mixer of this model keeps pages that could be held in 4 bits")
    for slot, request in paged:
        if not request.four_bit:
            raise UnsupportedError(f"cache slot {slot}: its mixer does not take pages of 4 bits")
    return kv_type


class CachePools:
    """Allocates the pools and the native manager for one engine.  ``kv_type``: None for pages of ``dtype``, "q4" for pages of
    4 bits (per cache slot codes and scales of the keys, then of the values, as ``ops.Q4Pages`` says)."""

    def __init__(self, cache_requests: Dict[int, object], *, page_size: int, num_pages, num_state_slots: int,
                 dtype: torch.dtype, device, reuse_prefixes: bool = False, kv_type: Optional[str] = None):
        self.kv_type = check_kv_type(kv_type, cache_requests)
        self.groups, self.states = plan_groups(cache_requests)
        self.page_size = int(page_size)
        self.dtype = dtype
        self.device = device
        if isinstance(num_pages, int):
            num_pages = [num_pages] * len(self.groups)
        if len(num_pages) != len(self.groups):
            raise InvalidArgumentError("one page count is needed for each group of layers")
        self.num_pages = [int(n) for n in num_pages]
        runtime = runtime_module()
        self.manager = runtime.CacheManager(
            [(self.page_size, pages, group.window or 0, group.keep_first)
             for group, pages in zip(self.groups, self.num_pages)],
            int(num_state_slots),
            # pages of a prompt prefix can be shared only where the pages are all a request keeps:
            # a mixer with a state of its own would have to store that state at every page's end
            bool(reuse_prefixes) and not self.states)
        self.pool_tensors: List[torch.Tensor] = []
        views: Dict[object, object] = {}
        # One page beyond those the manager hands out, per group: the scratch page.  No request
        # ever holds it; tokens that pad a captured step to its size class write there.
        self.scratch_pages: List[int] = list(self.num_pages)
        self.scratch_state_slot = int(num_state_slots)   # the spare row of every fixed-size state
        # Each pool lies between two guard regions of one page each, filled with a fixed word that
        # no kernel ever writes: `guards_intact()` (the tests call it after they ran) shows a write
        # that went past either end of a pool.
        self._guards: List[torch.Tensor] = []
        for index, (group, pages) in enumerate(zip(self.groups, self.num_pages)):
            rows = (pages + 1) * self.page_size * group.num_kv_heads     # key (or value) rows of one slot
            if self.kv_type == "q4":
                self._add_q4_group(index, group, pages, rows, views)
                continue
            count = len(group.slots) * rows * (group.head_dim + group.v_dim)
            guard = self.page_size * group.num_kv_heads * max(group.head_dim, group.v_dim)
            storage = torch.zeros(count + 2 * guard, dtype=dtype, device=device)
            storage[:guard].view(torch.int16 if storage.element_size() == 2 else torch.int32).fill_(GUARD_WORD)
            storage[guard + count:].view(torch.int16 if storage.element_size() == 2 else torch.int32).fill_(GUARD_WORD)
            self._guards.extend([storage[:guard], storage[guard + count:]])
            pool = storage[guard:guard + count]
            self.pool_tensors.append(pool)
            page_shape = (pages + 1, self.page_size, group.num_kv_heads)
            for position, slot in enumerate(group.slots):
                # a slot's keys, then its values: [slot][k | v][page][position][kv head][d or value size]
                base = position * rows * (group.head_dim + group.v_dim)
                k = pool[base:base + rows * group.head_dim].view(*page_shape, group.head_dim)
                v = pool[base + rows * group.head_dim:base + rows * (group.head_dim + group.v_dim)].view(
                    *page_shape, group.v_dim)
                views[slot] = PagedKVView(index, k, v, self.page_size, group.window, group.keep_first)
        for slot, request in self.states.items():
            # one row beyond the requests' own: the spare row, for entries that pad a captured step
            data = torch.zeros((int(num_state_slots) + 1, *request.shape), dtype=request.dtype, device=device)
            views[slot] = StateView(data)
        self._flat_views = views
        # what each cache slot of the schedule is handed: a view, or for a bundle a dict of views
        self.views: Dict[int, object] = {slot: bundle_views(request, slot, views)
                                         for slot, request in cache_requests.items() if request is not None}

    def _add_q4_group(self, index: int, group: CacheGroup, pages: int, rows: int, views: Dict[object, object]) -> None:
        def whole(count: int) -> int:
            return -(-count // _Q4_ALIGN) * _Q4_ALIGN

        code_bytes, scale_bytes = whole(rows * group.head_dim // 2), whole(rows * group.head_dim // Q4_GROUP * 2)
        count = len(group.slots) * 2 * (code_bytes + scale_bytes)
        guard = whole(self.page_size * group.num_kv_heads * group.head_dim)
        storage = torch.zeros(count + 2 * guard, dtype=torch.uint8, device=self.device)
        for region in (storage[:guard], storage[guard + count:]):
            region.view(torch.int16).fill_(GUARD_WORD)
            self._guards.append(region.view(torch.int16))
        pool = storage[guard:guard + count]
        self.pool_tensors.append(pool)
        shape = (pages + 1, group.num_kv_heads, self.page_size)
        for position, slot in enumerate(group.slots):
            tensors, at = [], position * 2 * (code_bytes + scale_bytes)
            for _ in range(2):                                   # keys, values
                tensors.append(pool[at:at + rows * group.head_dim // 2].view(*shape, group.head_dim // 2))
                at += code_bytes
                scales = pool[at:at + rows * group.head_dim // Q4_GROUP * 2].view(torch.bfloat16)
                tensors.append(scales.view(*shape, group.head_dim // Q4_GROUP))
                at += scale_bytes
            views[slot] = PagedQ4View(index, Q4Pages(*tensors), self.page_size, group.window, group.keep_first)

    def guards_intact(self) -> bool:
        """Whether the guard regions in front of and behind every pool still hold their word."""
        for guard in self._guards:
            words = guard.view(torch.int16 if guard.element_size() == 2 else torch.int32)
            if not bool((words == GUARD_WORD).all()):
                return False
        return True

    def audit(self) -> str:
        """"" when the manager's books are sound (no page lost, held twice or freed twice) and
        the guard regions are intact; else what is wrong."""
        problem = self.manager.audit()
        if not problem and not self.guards_intact():
            problem = "a guard region beside a cache pool was written"
        return problem

    def bytes(self) -> int:
        total = sum(p.numel() * p.element_size() for p in self.pool_tensors)
        for view in self._flat_views.values():
            if isinstance(view, StateView):
                total += view.data.numel() * view.data.element_size()
        return total

    def poison(self, value: float = float("nan")) -> None:
        """Fill every page with a value that shows when read (tests use NaN)."""
        if self.kv_type == "q4":
            for view in self._flat_views.values():
                if isinstance(view, PagedQ4View):    # a row of 4 bits shows the value through its scales
                    view.pages.k_scales.fill_(value)
                    view.pages.v_scales.fill_(value)
            return
        for pool in self.pool_tensors:
            pool.fill_(value)
