"""Page pools: which pages of a cache group are free, and who holds the others.

A page may have several holders (requests that were forked hold the full pages of their common
prefix together): it is free again when the last of them has given it back.

The free list is a stack (last freed, first taken), as the reference's allocator
(src/wllm/engine/kv_cache.py:27-54), so a page that a finished request gives back
is the next one handed out.  Unlike the reference, exhaustion is a typed exception
and giving back a page that is not held is an error instead of a silent clamp.
"""
from __future__ import annotations


class OutOfPages(RuntimeError):
    """A cache group has fewer free pages than a step needs."""

    def __init__(self, group: str, needed: int, free: int):
        super().__init__(f"cache group '{group}': {needed} pages needed, {free} free")
        self.group, self.needed, self.free = group, needed, free


class PagePool:
    def __init__(self, num_pages: int):
        if num_pages < 1:
            raise ValueError("a pool needs at least one page")
        self.num_pages = num_pages
        self._free = list(range(num_pages - 1, -1, -1))  # page 0 is taken first
        self._holders = [0] * num_pages
        self.takes = 0   # pages handed out so far; above num_pages means pages were used again

    @property
    def num_free(self) -> int:
        return len(self._free)

    def take(self) -> int:
        if not self._free:
            raise OutOfPages("?", 1, 0)
        page = self._free.pop()
        self._holders[page] = 1
        self.takes += 1
        return page

    def share(self, page: int) -> None:
        """One more holder of a page that is held."""
        if not self.is_held(page):
            raise RuntimeError(f"page {page} shared but not held")
        self._holders[page] += 1

    def give(self, page: int) -> bool:
        """One holder fewer; true when it was the last and the page is free."""
        if not self.is_held(page):
            raise RuntimeError(f"page {page} given back but not held (freed twice?)")
        self._holders[page] -= 1
        if self._holders[page]:
            return False
        self._free.append(page)
        return True

    def is_held(self, page: int) -> bool:
        return 0 <= page < self.num_pages and self._holders[page] > 0

    def holders(self, page: int) -> int:
        return self._holders[page] if 0 <= page < self.num_pages else 0

    def renumbered(self, num_pages: int) -> tuple:
        """(a pool of that many pages, {page here: page there}): the held pages are the new pool's first, in order, with the holders that they have here."""
        held = [p for p in range(self.num_pages) if self._holders[p]]
        if len(held) > num_pages:
            raise OutOfPages("?", len(held), num_pages)
        new = PagePool(num_pages)
        for p in held:
            new._holders[new._free.pop()] = self._holders[p]
        new.takes = self.takes
        return new, {p: i for i, p in enumerate(held)}
