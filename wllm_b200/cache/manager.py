"""The cache manager: pages of keys and values per group of layers, a block table per
request and group, and slots for per-request state of fixed size.

A *group* is a set of layers with the same needs: number of key/value heads, head
size and how much of the past they read (all of it, or a window).  Every group has
its own pool of pages and its own table per request; one page of a group holds
`page_size` tokens of all the group's layers.  Pages are taken when a step reserves
room for new tokens and given back when the request is closed, or, in a window
group, as soon as no later token can read them (the pages of the first `keep_first`
tokens of a sequence, which such a group may keep readable behind the window, stay).  Reserving for a step is atomic:
either every request of the step gets its pages or nothing changes and
`OutOfPages` is raised, which is how the scheduler learns that it has to preempt.

A request may be *forked*: the new one holds the full pages of the tokens that both have, together with the old one
(`PagePool` counts the holders), and a copy of the page that is partly written, so that nobody writes to a page that
somebody else reads.  Its per-request state is copied.  The whole cache may be given another number of pages
(`resize`): the live pages are moved to the front of new pools.

Beside the pages, every live request owns one *slot*: a row index into the state
tensors (per-request state of fixed size that a mixer may declare, for instance a
recurrent state) and, for the engine, a stable small integer for the request.
Gemma 1 declares no state; the slot is still taken and given back.

Reference for the bookkeeping this replaces: src/wllm/engine/kv_cache.py:63-303
(one table per sequence shared by all layers, reserve/advance, free_sequence).
Pool layout on the device, per group:
    [layer_in_group][k|v][page][kv_head][slot_in_page][head_dim]
A group whose value heads have a size of their own (`v_head_dim`) holds two pools of that layout
without the k|v axis, one for keys and one for values; a group whose values are the first elements of its
keys' rows (`values_in_keys`) holds the one pool of keys.  A window group may be one of blocks (`blocks`): a
token reads the earlier keys of its own block of `window` positions, so the pages in front of the block
that the next token lies in go back.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from ..kernels import ops
from .pages import OutOfPages, PagePool


@dataclass(frozen=True)
class CacheGroupSpec:
    name: str
    layers: int            # cache layers in the group
    kv_heads: int
    head_dim: int
    window: int | None = None   # None: every key is kept; n: a token reads the n latest keys (itself included)
    v_head_dim: int | None = None   # size of a value head when it differs from head_dim
    keep_first: int = 0             # with a window: the first keys of a sequence that stay readable behind it
    blocks: bool = False            # `window` is a block size: a token reads the earlier keys of its own block of positions
    values_in_keys: bool = False    # the values are the first v_head_dim elements of the keys' rows: one pool, no k|v axis

    def first_needed(self, num_tokens: int) -> int:
        """The oldest key that the token at position `num_tokens` (the next one) reads; every key for a group without a mask."""
        if self.window is None:
            return 0
        if self.blocks:
            return num_tokens - num_tokens % self.window
        return max(0, num_tokens - self.window + 1)


@dataclass(frozen=True)
class StateSpec:
    name: str
    shape: tuple
    dtype: torch.dtype = torch.float32


@dataclass
class RequestCache:
    """What one live request holds.  `tables[g][i]` is the page with tokens
    i*page_size .. (i+1)*page_size-1 in group g, or -1 once a window has passed it."""
    request_id: object
    slot: int
    tables: list
    num_tokens: int = 0        # tokens whose keys and values are written and committed
    reserved: int = 0          # tokens reserved by the step in flight
    closed: bool = False
    released_upto: list = field(default_factory=list)   # per group: pages below this index were given back
    version: int = 0           # bumped whenever a table changes (lets a reader cache a copy)
    forked: int = 0            # tokens that were in front of it when it was forked, or of a request forked from it: it may share pages below that


class CacheGroup:
    def __init__(self, spec: CacheGroupSpec, num_pages: int, page_size: int, dtype, device, poison: bool = False):
        self.spec = spec
        self.pool = PagePool(num_pages)
        self.page_size = page_size
        self.poison = poison
        self.dtype, self.device = dtype, device
        self.v_head_dim = spec.v_head_dim or spec.head_dim
        self._item = torch.empty((), dtype=dtype).element_size() if dtype is not None else 4
        self._allocate(num_pages)

    def _allocate(self, num_pages: int) -> None:
        spec, page_size, dtype, device = self.spec, self.page_size, self.dtype, self.device
        self.pages = None               # keys and values of one size: one pool with a k|v axis
        self.key_pages = self.value_pages = None      # value heads of their own size: two pools
        if device is not None:
            def pool(*shape):
                return torch.full(shape, float("nan"), dtype=dtype, device=device) if self.poison else \
                    torch.zeros(shape, dtype=dtype, device=device)
            if spec.values_in_keys:
                self.key_pages = self.value_pages = pool(spec.layers, num_pages, spec.kv_heads, page_size, spec.head_dim)
            elif self.v_head_dim == spec.head_dim:
                self.pages = pool(spec.layers, 2, num_pages, spec.kv_heads, page_size, spec.head_dim)
            else:
                self.key_pages = pool(spec.layers, num_pages, spec.kv_heads, page_size, spec.head_dim)
                self.value_pages = pool(spec.layers, num_pages, spec.kv_heads, page_size, self.v_head_dim)
        # a layer's keys and values as views, made once (the pools stay where they are)
        self._views = [(self.pages[i, 0], self.pages[i, 1]) if self.pages is not None else (self.key_pages[i], self.value_pages[i])
                       for i in range(spec.layers)] if device is not None else []

    def tensors(self) -> list:
        """The pools, [layers, (k | v,) pages, kv heads, slots, head]."""
        return [t for t in (self.pages, self.key_pages, None if self.spec.values_in_keys else self.value_pages) if t is not None]

    def give(self, pages: list) -> None:
        """Pages go back to the pool, or lose a holder; with `poison` the contents of those that are free now become NaN (in
        stream order, so a step still running has read them before)."""
        freed = [page for page in pages if self.pool.give(page)]
        if self.poison and freed:
            for pool in self.tensors():
                pool.index_fill_(pool.dim() - 4, torch.tensor(freed, dtype=torch.long, device=pool.device), float("nan"))

    def resize(self, num_pages: int) -> dict:
        """New pools of that many pages; the held pages move to their front.  {page before: page now}"""
        try:
            pool, moved = self.pool.renumbered(num_pages)
        except OutOfPages as e:
            raise OutOfPages(self.spec.name, e.needed, e.free) from None
        old = self.tensors()
        before = (self.pages, self.key_pages, self.value_pages, self._views)
        try:
            self._allocate(num_pages)
            if moved and old:
                ops.copy_pages([(a, b, list(moved), list(moved.values()), None) for a, b in zip(old, self.tensors())])
        except BaseException:
            self.pages, self.key_pages, self.value_pages, self._views = before
            raise
        self.pool = pool
        return moved

    def keys(self, layer: int) -> torch.Tensor:
        return self._views[layer][0]

    def values(self, layer: int) -> torch.Tensor:
        return self._views[layer][1]

    def bytes_per_token(self) -> int:
        per_head = self.spec.head_dim if self.spec.values_in_keys else self.spec.head_dim + self.v_head_dim
        return self.spec.layers * self.spec.kv_heads * per_head * self._item


class StateSlots:
    """Rows of fixed-size per-request state: tensor `name` has shape [num_slots, *shape].  `spare`: more slots beside those of the requests, for prefixes that are kept; there
    are none where a slot is memory."""

    def __init__(self, num_slots: int, specs: list, device, spare: int = 0):
        self.num_slots, self.specs = num_slots, list(specs)
        self.total = num_slots + (0 if self.specs else spare)
        self._free = list(range(self.total - 1, -1, -1))
        self._held = [False] * self.total
        self.tensors = {}
        if device is not None:
            for s in specs:
                self.tensors[s.name] = torch.zeros((num_slots,) + tuple(s.shape), dtype=s.dtype, device=device)

    @property
    def num_free(self) -> int:
        """Requests that may still take one."""
        return min(self.num_slots, len(self._free))

    def take(self, zero: bool = True) -> int:
        if not self._free:
            raise OutOfPages("request slots", 1, 0)
        slot = self._free.pop()
        self._held[slot] = True
        for t in self.tensors.values() if zero else ():   # a new request starts from zero state
            t[slot].zero_()
        return slot

    def rows(self) -> list:
        """The state tensors as pools of pages of one slot."""
        return [t.view(self.num_slots, 1, 1, -1) for t in self.tensors.values() if t.numel()]

    def give(self, slot: int) -> None:
        if not self._held[slot]:
            raise RuntimeError(f"state slot {slot} given back but not held")
        self._held[slot] = False
        self._free.append(slot)


class CacheManager:
    def __init__(self, groups: list, page_size: int, num_pages: int, max_requests: int, states: list = (),
                 dtype=torch.bfloat16, device=None, poison: bool = False, prefix_slots: int = 0):
        """`prefix_slots`: slots beside those of `max_requests` requests, for prefixes (none if there is per-request state, where they take the requests').  `poison` (a debugging aid; the tests switch it on): pools start as NaN instead of zeros and every
        page is filled with NaN again when it is given back, so a kernel that reads a slot that was never
        written, or a page that its request no longer holds, shows at once in the logits."""
        if page_size < 1:
            raise ValueError("page_size must be positive")
        self.page_size = page_size
        self.groups = [CacheGroup(g, num_pages, page_size, dtype, device, poison) for g in groups]
        self.slots = StateSlots(max_requests, list(states), device, prefix_slots)
        self.live: dict = {}
        self.dtype, self.device = dtype, device
        self.pages_high_water = [0] * len(self.groups)

    # -- requests ------------------------------------------------------------------
    def open(self, request_id) -> RequestCache:
        if request_id in self.live:
            raise KeyError(f"request {request_id!r} is already open")
        rc = RequestCache(request_id, self.slots.take(), [[] for _ in self.groups],
                          released_upto=[0] * len(self.groups))
        self.live[request_id] = rc
        return rc

    def fork(self, rc: RequestCache, request_id, num_tokens: int | None = None) -> RequestCache:
        """A new request that begins with the first `num_tokens` committed tokens of `rc` (None: all of them): it holds their full
        pages together with it, and gets a copy of the page that the last of them lie in and of the per-request state.  One page
        of every group where num_tokens is no whole number of pages, and a slot; `OutOfPages` leaves everything as it was.  Per-request
        state is that of all tokens, so a cache that has some forks at all of them; and a window must not have passed what the
        token behind the first `num_tokens` reads."""
        n = rc.num_tokens if num_tokens is None else num_tokens
        if rc.closed or rc.reserved:
            raise RuntimeError(f"request {rc.request_id!r} is " + ("closed" if rc.closed else "in a step"))
        if not 0 <= n <= rc.num_tokens:
            raise ValueError(f"request {rc.request_id!r} has {rc.num_tokens} tokens; it cannot be forked at {n}")
        if n != rc.num_tokens and self.slots.specs:
            raise ValueError(f"request {rc.request_id!r} has state of all its {rc.num_tokens} tokens; it cannot be forked at {n}")
        if request_id in self.live:
            raise KeyError(f"request {request_id!r} is already open")
        ps = self.page_size
        full, tail = n // ps, n % ps
        for g, table in zip(self.groups, rc.tables):
            seen = list(range(min(g.spec.first_needed(n), n) // ps, -(-n // ps)))
            if g.spec.window is not None:
                seen += range(min(-(-g.spec.keep_first // ps), -(-n // ps)))
            if any(table[i] < 0 for i in seen):
                raise ValueError(f"request {rc.request_id!r}: the window of group '{g.spec.name}' has passed tokens that are read behind the first {n}")
            if tail and g.pool.num_free < 1:
                raise OutOfPages(g.spec.name, 1, 0)
        new = RequestCache(request_id, self.slots.take(zero=False), [], num_tokens=n, released_upto=[min(u, full) for u in rc.released_upto])
        moves = []
        for g, table in zip(self.groups, rc.tables):
            mine = list(table[:full])
            for page in mine:
                if page >= 0:
                    g.pool.share(page)
            if tail:
                mine.append(g.pool.take())
                moves += [(t, t, [table[full]], [mine[-1]], [tail]) for t in g.tensors()]
            new.tables.append(mine)
        moves += [(t, t, [rc.slot], [new.slot], None) for t in self.slots.rows()]
        try:
            for i in range(0, len(moves), ops.MAX_COPY_POOLS):
                ops.copy_pages(moves[i:i + ops.MAX_COPY_POOLS])
        except BaseException:
            for g, mine in zip(self.groups, new.tables):
                g.give([page for page in mine if page >= 0])
            self.slots.give(new.slot)
            raise
        rc.forked, new.forked = max(rc.forked, n), n
        self.live[request_id] = new
        self._note_high_water()
        return new

    def resize(self, num_pages: int) -> None:
        """Another number of pages in every group, with the live pages at the front of the new pools (every table follows; whoever holds views
        of the old pools asks for them again).  `OutOfPages` if some group holds more than that, and everything is as it was."""
        if num_pages < 1:
            raise ValueError("a pool needs at least one page")
        for rc in self.live.values():
            if rc.reserved:
                raise RuntimeError(f"request {rc.request_id!r} is in a step")
        for g in self.groups:
            if g.pool.num_pages - g.pool.num_free > num_pages:
                raise OutOfPages(g.spec.name, g.pool.num_pages - g.pool.num_free, num_pages)
        for gi, g in enumerate(self.groups):
            moved = g.resize(num_pages)
            for rc in self.live.values():
                rc.tables[gi] = [page if page < 0 else moved[page] for page in rc.tables[gi]]
                rc.version += 1

    def close(self, rc: RequestCache) -> None:
        """Give back everything the request holds.  Closing twice is an error."""
        if rc.closed:
            raise RuntimeError(f"request {rc.request_id!r} closed twice")
        for g, table in zip(self.groups, rc.tables):
            g.give([page for page in reversed(table) if page >= 0])
            table.clear()
        self.slots.give(rc.slot)
        rc.closed = True
        del self.live[rc.request_id]

    # -- pages ---------------------------------------------------------------------
    def _pages_for(self, rc: RequestCache, extra: int) -> int:
        total = rc.num_tokens + rc.reserved + extra
        return -(-total // self.page_size)

    def pages_needed(self, wants: list) -> list:
        """Pages that each group must hand out so that every (request, n_new) of `wants` fits."""
        need = [0] * len(self.groups)
        for rc, n in wants:
            target = self._pages_for(rc, n)
            for gi in range(len(self.groups)):
                need[gi] += max(0, target - len(rc.tables[gi]))
        return need

    def can_reserve(self, wants: list) -> bool:
        return all(n <= g.pool.num_free for n, g in zip(self.pages_needed(wants), self.groups))

    def reserve(self, wants: list) -> None:
        """Take the pages for all of `wants` = [(request, n_new_tokens)], or none of them."""
        need = self.pages_needed(wants)
        for n, g in zip(need, self.groups):
            if n > g.pool.num_free:
                raise OutOfPages(g.spec.name, n, g.pool.num_free)
        for rc, n in wants:
            if rc.closed:
                raise RuntimeError(f"request {rc.request_id!r} is closed")
            target = self._pages_for(rc, n)
            for g, table in zip(self.groups, rc.tables):
                while len(table) < target:
                    table.append(g.pool.take())
                    rc.version += 1
            rc.reserved += n
        self._note_high_water()

    def _note_high_water(self) -> None:
        for gi, g in enumerate(self.groups):
            used = g.pool.num_pages - g.pool.num_free
            self.pages_high_water[gi] = max(self.pages_high_water[gi], used)

    def token_slots(self, rc: RequestCache, group: int, start: int, n: int) -> list:
        """Flat slots (page * page_size + offset) of the tokens start .. start+n-1 of a request."""
        table, ps = rc.tables[group], self.page_size
        return [table[p // ps] * ps + p % ps for p in range(start, start + n)]

    def commit(self, rc: RequestCache, n: int) -> None:
        """The step wrote `n` reserved tokens.  Window groups give back the pages that
        no later token can read: a token at position p reads keys p-window+1 .. p."""
        if n > rc.reserved:
            raise RuntimeError("commit of more tokens than reserved")
        rc.reserved -= n
        rc.num_tokens += n
        for gi, g in enumerate(self.groups):
            w = g.spec.window
            if w is None:
                continue
            first_needed = g.spec.first_needed(rc.num_tokens)      # oldest key the next token reads
            upto = min(max(0, first_needed // self.page_size), len(rc.tables[gi]))
            kept = -(-g.spec.keep_first // self.page_size)       # pages that hold a sequence's kept first keys stay
            passed = list(range(max(rc.released_upto[gi], kept), upto))
            g.give([rc.tables[gi][i] for i in passed])
            for i in passed:
                rc.tables[gi][i] = -1
                rc.version += 1
            rc.released_upto[gi] = max(rc.released_upto[gi], upto)

    def cancel_reservation(self, rc: RequestCache) -> None:
        """Undo a reservation that no step used: surplus pages go back."""
        rc.reserved = 0
        target = -(-rc.num_tokens // self.page_size)
        for g, table in zip(self.groups, rc.tables):
            surplus = []
            while len(table) > target:
                page = table.pop()
                rc.version += 1
                if page >= 0:          # (a window never passes a page that holds no committed token; checked all the same)
                    surplus.append(page)
            g.give(surplus)

    # -- figures -------------------------------------------------------------------
    def free_pages(self) -> list:
        return [g.pool.num_free for g in self.groups]

    def bytes_per_token(self) -> int:
        return sum(g.bytes_per_token() for g in self.groups)

    def check(self) -> None:
        """Every page is either free or in as many live tables as it has holders, at the same place and behind the same pages in all of them,
        and no slot behind the tokens that its holders have in common is written by more than one of them; used by the tests."""
        for gi, g in enumerate(self.groups):
            seen = {}
            for rc in self.live.values():
                for i, page in enumerate(rc.tables[gi]):
                    if page < 0:
                        continue
                    if not g.pool.is_held(page):
                        raise AssertionError(f"group {g.spec.name}: page {page} is in a table but free")
                    seen.setdefault(page, []).append((i, rc))
            for page, held in seen.items():
                who = [rc.request_id for _, rc in held]
                if len(held) != g.pool.holders(page):
                    raise AssertionError(f"group {g.spec.name}: page {page} held by {who!r}, counted {g.pool.holders(page)} times")
                if len(held) > 1 and (len({i for i, _ in held}) > 1 or any((i + 1) * self.page_size > min(rc.num_tokens, rc.forked) for i, rc in held)):
                    raise AssertionError(f"group {g.spec.name}: page {page} held by {who!r} at places where they do not agree")
            if len(seen) + g.pool.num_free != g.pool.num_pages:
                raise AssertionError(f"group {g.spec.name}: {g.pool.num_pages - g.pool.num_free - len(seen)} pages lost")
