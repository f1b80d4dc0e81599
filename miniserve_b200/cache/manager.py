"""The cache manager: pages of keys and values in groups, block tables per request, and
slots for per-request state of fixed size.

The reference keeps one pool tensor for all layers and one table per request
(miniserve/cache/kv_pool.py:14-50, miniserve/cache/kv_cache.py:33-136 with the prefix cache
switched off). Here run entries with the same need (kv heads, head size, window) form a
*group*; each group has pages, an allocator and per-request tables of its own, because a group
that only looks a window back gives pages back while a request is still running, and a group
that keeps every key does not. Pages return to their allocator when a request ends or is
preempted (``release``), when an admission is refused, and, for a windowed group, as soon as
the window has passed them (``trim``). A failed ``reserve`` changes nothing.

Beside the pages there are slots for per-request state of fixed size: one slot id per live
request, indexing a tensor per run entry that declared such state. Qwen3 declares none, so
the tensors are absent and only the slot ids are handed out.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Sequence

import torch

from ..ops.cache8 import Pool8, read_cache, takes
from ..parts.base import FixedState, PagedKV, flat_needs
from ..parts.decoder import EntryCache
from .blocks import BlockAllocator, BlockTable, OutOfBlocks


@dataclass
class CacheGroup:
    need: PagedKV
    entries: list[int]  # run entries that own a cache in this group
    allocator: BlockAllocator
    page_size: int
    k: torch.Tensor | None = None  # [entries, pages + 1, kv_heads, page_size, head_dim]; in 8 bits the codes
    v: torch.Tensor | None = None
    k_exponents: torch.Tensor | None = None  # in 8 bits: [entries, pages + 1, kv_heads, page_size]
    v_exponents: torch.Tensor | None = None
    eight_bits: bool = False

    @property
    def pad_page(self) -> int:
        """A page outside the allocator, written and read only by padding rows."""
        return self.allocator.num_blocks

    def bytes_per_token(self, itemsize: int) -> int:
        vector = vector_bytes(self.need.head_dim, itemsize, self.eight_bits)
        return (2 if self.need.values else 1) * len(self.entries) * self.need.kv_heads * vector

    def pools(self, index: int) -> tuple:
        """The pools of keys and values of the group's entry ``index``."""
        if self.k is None:
            return None, None
        if self.eight_bits:
            return Pool8(self.k[index], self.k_exponents[index]), Pool8(self.v[index], self.v_exponents[index])
        return self.k[index], self.v[index]


@dataclass
class KVEntryView:
    """What an attention mixer gets: its group's index (to pick the page table from the step
    context), its own K and V pools [pages + 1, kv_heads, page_size, head_dim] (``Pool8`` where they are in 8 bits)."""

    group: int
    k: "torch.Tensor | Pool8 | None"
    v: "torch.Tensor | Pool8 | None"
    page_size: int


@dataclass
class StateEntryView:
    """What a mixer with fixed-size state gets: ``state[slot]`` belongs to the request whose
    slot id is ``ctx.state_slot[row]``. The tensor has one slot more than the cache has requests:
    the padding rows of a captured graph carry that slot's id, so a mixer needs no mask for them."""

    state: torch.Tensor | None
    shape: tuple[int, ...]


@dataclass
class RequestCache:
    """Everything one live request holds: a table per group and a state slot."""

    tables: list[BlockTable]
    state_slot: int = -1
    released: bool = False

    @property
    def num_tokens(self) -> int:
        return self.tables[0].num_tokens if self.tables else self._tokens_without_tables

    _tokens_without_tables: int = 0


def group_needs(entry_caches: Sequence[EntryCache]) -> tuple[list[tuple[PagedKV, int]], list[FixedState]]:
    """What a model's run entries ask of the cache: ``[(need, number of entries)]`` for the paged
    groups (entries with equal needs share a group), and the fixed-size states, one per owning
    entry. The order of the groups is the one ``CacheManager`` uses."""
    groups: dict[PagedKV, int] = {}
    states: list[FixedState] = []
    for i, ec in enumerate(entry_caches):
        if ec.owner != i:
            continue
        for need in flat_needs(ec.need):  # a mixer made of several may need pages and state, or several states
            if isinstance(need, PagedKV):
                groups[need] = groups.get(need, 0) + 1
            elif isinstance(need, FixedState):
                states.append(need)
    return list(groups.items()), states


def window_pages(window: int, page_size: int, step_tokens: int) -> int:
    """The most pages a request holds in a group that looks ``window`` keys back, when a step brings
    it at most ``step_tokens`` tokens: the window and the step's tokens (pages are given back after
    the step), plus the pages both ends cut into."""
    return -(-(window + step_tokens) // page_size) + 1


def vector_bytes(head_dim: int, itemsize: int, eight_bits: bool) -> int:
    """Bytes of one head's vector in the cache: its numbers, or a code each and an exponent."""
    return head_dim + 1 if eight_bits else head_dim * itemsize


def check_needs8(entry_caches: Sequence[EntryCache], page_size: int) -> None:
    """Raise unless what the run entries ask of the cache can be held in 8 bits."""
    for need, _ in group_needs(entry_caches)[0]:
        if not need.values:
            raise ValueError("an 8-bit cache holds keys and values, not one latent vector for both")
        if not takes(need.head_dim, page_size):
            raise ValueError(f"an 8-bit cache takes head sizes that are multiples of 16 up to 256 and pages of a power of two of at least 8 tokens, not "
                             f"{need.head_dim} and {page_size}")


KV_DTYPES = ("auto", "fp8")  # how keys and values are held: in the model's type, or in 8 bits (``ops.Pool8``)


class CacheManager:
    def __init__(self, entry_caches: Sequence[EntryCache], num_pages: "int | Sequence[int]", page_size: int, max_requests: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None,
                 poison: bool = False, poison_on_free: bool = False, step_tokens: int | None = None, kv_dtype: str = "auto"):
        """``entry_caches``: one per run entry (``DecoderModel.entry_caches``). ``num_pages``:
        pages of ``page_size`` tokens, one number for every group or one per group (in the order
        of ``group_needs``). ``device`` None keeps everything on the host (bookkeeping only, for
        tests). ``poison`` fills the pools with NaN so that a read of a slot nobody wrote shows
        up; ``poison_on_free`` also fills a request's pages with NaN when it gives them back, so
        that a stale key read through a reused page shows up (a debugging aid: it launches a fill
        per release). ``step_tokens``: the most tokens a step brings one request; with it,
        ``pages_for`` knows that a windowed group never holds a whole long request. ``kv_dtype``: "fp8" keeps keys and
        values in 8 bits (per-request state of fixed size stays as it is)."""
        if kv_dtype not in KV_DTYPES:
            raise ValueError(f"kv_dtype is one of {KV_DTYPES}, not {kv_dtype!r}")
        eight_bits = kv_dtype == "fp8"
        if eight_bits:
            check_needs8(entry_caches, page_size)
            if dtype != torch.bfloat16:
                raise ValueError(f"an 8-bit cache belongs to a bfloat16 model, not to one in {dtype}")
        self.kv_dtype = kv_dtype
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two, got {page_size}")
        needs, _ = group_needs(entry_caches)
        per_group = [int(num_pages)] * len(needs) if isinstance(num_pages, int) else [int(n) for n in num_pages]
        if len(per_group) != len(needs):
            raise ValueError(f"{len(per_group)} page counts for {len(needs)} cache groups")
        if any(n < 1 for n in per_group) or (isinstance(num_pages, int) and num_pages < 1):
            raise ValueError(f"the pool needs at least one page, got {num_pages}")
        self.page_size = page_size
        self.num_pages = max(per_group) if per_group else (num_pages if isinstance(num_pages, int) else 0)
        self.step_tokens = step_tokens
        self.poison_on_free = poison_on_free
        self.max_requests = max_requests
        self.dtype = dtype
        self.device = torch.device(device) if device is not None else None
        self.groups: list[CacheGroup] = []
        self._entry_view: list[KVEntryView | StateEntryView | None] = []
        self._state_entries: list[tuple[int, FixedState]] = []
        by_need: dict[PagedKV, int] = {}
        owners: dict[tuple[int, int], tuple[int, int]] = {}  # (owner entry, which of its needs) -> (group, index in group)
        for i, ec in enumerate(entry_caches):
            if ec.owner != i or ec.need is None:
                continue
            for n, need in enumerate(flat_needs(ec.need)):
                if isinstance(need, PagedKV):
                    g = by_need.get(need)
                    if g is None:
                        g = len(self.groups)
                        by_need[need] = g
                        self.groups.append(CacheGroup(need, [], BlockAllocator(per_group[g], page_size), page_size, eight_bits=eight_bits))
                    owners[(i, n)] = (g, len(self.groups[g].entries))
                    self.groups[g].entries.append(i)
                elif isinstance(need, FixedState):
                    self._state_entries.append(((i, n), need))
                else:
                    raise TypeError(f"run entry {i} asks for an unknown kind of cache: {need!r}")
        if self.device is not None:
            for grp in self.groups:
                shape = (len(grp.entries), grp.allocator.num_blocks + 1, grp.need.kv_heads, page_size, grp.need.head_dim)
                if eight_bits:
                    grp.k, grp.v = (torch.full(shape, 0x7F if poison else 0, dtype=torch.uint8, device=self.device) for _ in range(2))
                    grp.k_exponents, grp.v_exponents = (torch.full(shape[:-1], 255 if poison else 0, dtype=torch.uint8, device=self.device) for _ in range(2))
                    continue
                fill = float("nan") if poison else 0.0
                grp.k = torch.full(shape, fill, dtype=dtype, device=self.device)
                grp.v = torch.full(shape, fill, dtype=dtype, device=self.device) if grp.need.values else grp.k
        state_tensors: dict[tuple[int, int], torch.Tensor | None] = {}
        for i, need in self._state_entries:
            # one slot more than there are requests: the padding rows of a captured graph read and write it
            state_tensors[i] = (torch.zeros((max_requests + 1, *need.shape), dtype=need.dtype, device=self.device)
                                if self.device is not None else None)
        def view(owner: int, need, count: list):
            """The view of one need, or a tuple of views shaped like a tuple of needs."""
            if need is None:
                return None
            if not isinstance(need, (PagedKV, FixedState)):
                return tuple(view(owner, part, count) for part in need)
            n = count[0]
            count[0] += 1
            if isinstance(need, PagedKV):
                g, idx = owners[(owner, n)]
                grp = self.groups[g]
                return KVEntryView(g, *grp.pools(idx), page_size)
            return StateEntryView(state_tensors[(owner, n)], tuple(need.shape))

        def merged(own, other):
            """``own`` with ``other``'s views where it has none (an entry that reads part of its cache from another)."""
            if own is None:
                return other
            if isinstance(own, tuple) and isinstance(other, tuple) and len(own) == len(other):
                return tuple(merged(a, b) for a, b in zip(own, other))
            return own

        for ec in entry_caches:
            v = view(ec.owner, ec.need, [0])
            shares = getattr(ec, "shares", None)
            self._entry_view.append(v if shares is None else merged(v, self._entry_view[shares]))
        self._state_views = [v for v in self._flat_views() if isinstance(v, StateEntryView)]
        self._free_slots = list(range(max_requests - 1, -1, -1))
        self._live: set[int] = set()

    # ------------------------------------------------------------------ views and sizes
    @property
    def pad_state_slot(self) -> int:
        """A state slot outside the ones requests get, for padding rows (as ``pad_page`` is for pages)."""
        return self.max_requests

    @property
    def entry_views(self) -> list:
        return self._entry_view

    @property
    def num_groups(self) -> int:
        return len(self.groups)

    def bytes_per_token(self) -> int:
        item = torch.empty((), dtype=self.dtype).element_size()
        return sum(g.bytes_per_token(item) for g in self.groups)

    def pool_bytes(self) -> int:
        return sum((g.k.numel() * g.k.element_size() + (g.k_exponents.numel() if g.eight_bits else 0)) * (2 if g.need.values else 1)
                   for g in self.groups if g.k is not None)

    def state_bytes(self) -> int:
        """Bytes of the per-request state tensors (one slot per request the cache can hold)."""
        seen = {id(v.state): v.state for v in self._state_views if v.state is not None}
        return sum(t.numel() * t.element_size() for t in seen.values())

    def _flat_views(self) -> list:
        out: list = []

        def walk(v):
            if isinstance(v, tuple):
                for part in v:
                    walk(part)
            elif v is not None:
                out.append(v)

        for v in self._entry_view:
            walk(v)
        return out

    def state_tensors(self) -> list[torch.Tensor]:
        """Every per-request state tensor once (slot-indexed along the first axis)."""
        seen = {id(v.state): v.state for v in self._state_views if v.state is not None}
        return list(seen.values())

    # ------------------------------------------------------------------ requests
    def new_request(self) -> RequestCache:
        """Empty tables and a state slot for a request that is being admitted."""
        if not self._free_slots:
            raise OutOfBlocks(f"all {self.max_requests} request slots are taken")
        slot = self._free_slots.pop()
        self._live.add(slot)
        return RequestCache([g.allocator.new_table() for g in self.groups], slot)

    def release(self, rc: RequestCache) -> None:
        """Give back everything ``rc`` holds (request finished, aborted, preempted or refused)."""
        if rc.released:
            raise ValueError("request cache released twice")
        if self.poison_on_free and self.device is not None:
            for g, t in zip(self.groups, rc.tables):
                held = [b for b in t.blocks if b >= 0]
                if held and g.k is not None:
                    idx = torch.tensor(held, dtype=torch.long, device=self.device)
                    if g.eight_bits:
                        g.k[:, idx] = g.v[:, idx] = 0x7F
                        g.k_exponents[:, idx] = g.v_exponents[:, idx] = 255
                        continue
                    g.k[:, idx] = float("nan")
                    g.v[:, idx] = float("nan")
        for t in rc.tables:
            t.release()
        if rc.state_slot >= 0:
            self._live.discard(rc.state_slot)
            self._free_slots.append(rc.state_slot)
        rc.state_slot = -1
        rc.released = True

    def read(self, rc: RequestCache, entry: int, start: int = 0, stop: int | None = None, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values that run entry ``entry`` has cached for a request, positions [start, stop) (default: all), as
        dense rows [n, kv_heads, head_dim] in ``dtype`` (default: the model's): behind norm and rotation, as attention reads them."""
        if rc.released:
            raise ValueError("read of a released request cache")
        view = self._entry_view[entry]
        if not isinstance(view, KVEntryView):
            raise ValueError(f"run entry {entry} has no single cache of keys and values")
        if view.k is None:
            raise ValueError("read of a cache that keeps books alone: it has no pools")
        table = rc.tables[view.group]
        stop = table.num_tokens if stop is None else stop
        if not 0 <= start <= stop <= table.num_tokens:
            raise ValueError(f"positions [{start}, {stop}) of a request of {table.num_tokens} tokens")
        blocks = table.blocks
        if any(b < 0 for b in blocks[start // self.page_size:-(-stop // self.page_size)]):
            raise ValueError(f"positions [{start}, {stop}) have left the window: their pages were given back")
        dtype = dtype or self.dtype
        n, shape = stop - start, view.k.shape
        if not isinstance(view.k, Pool8):
            pos = torch.arange(start, stop, device=self.device)
            page = torch.tensor(blocks, dtype=torch.long, device=self.device)[pos // self.page_size]
            return view.k[page, :, pos % self.page_size].to(dtype), view.v[page, :, pos % self.page_size].to(dtype)
        k, v = (torch.empty((n, shape[1], shape[3]), dtype=dtype, device=self.device) for _ in range(2))
        if n:
            i32 = dict(dtype=torch.int32, device=self.device)
            read_cache(k, v, view.k, view.v, torch.arange(start, stop, **i32), torch.zeros(n, **i32), torch.tensor([0, len(blocks)], **i32),
                       torch.tensor(blocks, **i32), torch.zeros(1, **i32))
        return k, v

    @property
    def num_free_slots(self) -> int:
        return len(self._free_slots)

    # ------------------------------------------------------------------ page budget
    def num_free(self) -> tuple[int, ...]:
        return tuple(g.allocator.num_free for g in self.groups)

    def pages_for(self, num_tokens: int) -> tuple[int, ...]:
        """Pages per group that a request of ``num_tokens`` tokens may hold at its largest: all of
        them, or, in a windowed group (when the step size is known), the window and a step's tokens."""
        out = []
        for g in self.groups:
            n = -(-num_tokens // g.page_size)
            if g.need.window and self.step_tokens:
                n = min(n, window_pages(g.need.window, g.page_size, self.step_tokens))
            out.append(n)
        return tuple(out)

    def group_pages(self) -> tuple[int, ...]:
        """Pages each group's pool has."""
        return tuple(g.allocator.num_blocks for g in self.groups)

    def pages_needed(self, rc: RequestCache, new_tokens: int) -> tuple[int, ...]:
        """Pages per group that appending ``new_tokens`` to ``rc`` would allocate."""
        return tuple(t.blocks_needed(new_tokens) for t in rc.tables)

    def pages_held(self, rc: RequestCache) -> tuple[int, ...]:
        """Pages per group that ``rc`` holds now (a windowed group has given the older ones back)."""
        return tuple(t.num_blocks for t in rc.tables)

    def pages_outstanding(self, rc: RequestCache, upto_tokens: int) -> tuple[int, ...]:
        """Pages per group that ``rc`` may still take, net of what it gives back, before its
        sequence reaches ``upto_tokens`` tokens: the pages not yet allocated, but in a windowed
        group (when the step size is known) no more than brings it to the most it ever holds."""
        out = []
        for g, t in zip(self.groups, rc.tables):
            n = max(0, -(-upto_tokens // g.page_size) - t.num_entries)
            if g.need.window and self.step_tokens:
                n = min(n, max(0, window_pages(g.need.window, g.page_size, self.step_tokens) - t.num_blocks))
            out.append(n)
        return tuple(out)

    def fits(self, need: Sequence[int], margin: Sequence[int] | None = None) -> bool:
        free = self.num_free()
        margin = margin or (0,) * len(free)
        return all(n <= f - m for n, f, m in zip(need, free, margin))

    def reserve(self, rows: Sequence[tuple[RequestCache, int]]) -> None:
        """Extend every row's tables by its new tokens. All or nothing: if any group is short,
        raise ``OutOfBlocks`` with every table as it was (miniserve/engine/model_runner.py:309-315)."""
        for gi, g in enumerate(self.groups):
            need = sum(rc.tables[gi].blocks_needed(n) for rc, n in rows)
            if need > g.allocator.num_free:
                raise OutOfBlocks(f"need {need} free pages in cache group {gi}, {g.allocator.num_free} free")
        for rc, n in rows:
            if rc.released:
                raise ValueError("reserve on a released request cache")
            for t in rc.tables:
                t.append_tokens(n)
            rc._tokens_without_tables += n

    def trim(self, rc: RequestCache) -> int:
        """After a step: give back the pages of windowed groups that no later query can reach.
        The next query sits at position ``num_tokens`` and sees keys from
        ``num_tokens - window + 1`` on. Returns the number of pages freed."""
        freed = 0
        for g, t in zip(self.groups, rc.tables):
            if g.need.window:
                freed += t.release_below(t.num_tokens - g.need.window + 1)
        return freed

    # ------------------------------------------------------------------ checks
    def check_invariants(self) -> None:
        for g in self.groups:
            g.allocator.check_invariants()
        assert len(set(self._free_slots)) == len(self._free_slots), "a state slot is free twice"
        assert not (set(self._free_slots) & self._live), "a state slot is both free and live"
        assert len(self._free_slots) + len(self._live) == self.max_requests, "a state slot was lost"

    def is_idle(self) -> bool:
        """Nothing held by anyone: every page and every slot is free."""
        return all(g.allocator.num_free == g.allocator.num_blocks for g in self.groups) and not self._live
