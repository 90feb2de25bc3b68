"""Page and slot pools: plain host bookkeeping, no device memory.

The reference's ``BlockPool`` is a LIFO free list with reference counts
(``pkg/inference/paged_kvcache.go:34-117``).  Pages here count their holders too: one, unless
a request was forked; the pool refuses a page that is freed more often than it is held.
"""
from __future__ import annotations

from typing import Dict, List


class OutOfPages(RuntimeError):
    """The pool cannot give as many pages as were asked for; nothing was taken."""


class OutOfSlots(RuntimeError):
    """Every per-request state slot is in use."""


class PagePool:
    def __init__(self, num_pages: int):
        if num_pages < 0:
            raise ValueError("num_pages must be >= 0")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages - 1, -1, -1))   # pop() gives page 0 first
        self._holders = [0] * num_pages

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self, n: int) -> List[int]:
        """``n`` pages, all or none."""
        if n > len(self._free):
            raise OutOfPages(f"asked for {n} pages, {len(self._free)} of {self.num_pages} free")
        out = [self._free.pop() for _ in range(n)]
        for p in out:
            self._holders[p] = 1
        return out

    def share(self, page: int) -> None:
        """One more holder of a page that is held."""
        if not (0 <= page < self.num_pages) or not self._holders[page]:
            raise ValueError(f"page {page} is not held: it cannot be shared")
        self._holders[page] += 1

    def holders(self, page: int) -> int:
        return self._holders[page]

    def give_back(self, page: int) -> None:
        if not (0 <= page < self.num_pages):
            raise ValueError(f"page {page} is not of this pool (0..{self.num_pages - 1})")
        if not self._holders[page]:
            raise RuntimeError(f"page {page} freed twice")
        self._holders[page] -= 1
        if not self._holders[page]:
            self._free.append(page)

    def held_pages(self) -> List[int]:
        return [p for p, h in enumerate(self._holders) if h]

    def compact(self) -> Dict[int, int]:
        """Renumber: the held pages become the lowest ones.  Returns the moves, old number -> new number (a held page to one that was
        free); the caller moves the contents and renames the pages in its tables."""
        held = self.held_pages()
        gaps = [p for p in range(len(held)) if not self._holders[p]]
        moves = dict(zip((p for p in held if p >= len(held)), gaps))
        for old, new in moves.items():
            self._holders[new], self._holders[old] = self._holders[old], 0
        self._free = list(range(self.num_pages - 1, len(held) - 1, -1))
        return moves


class SlotPool(PagePool):
    """Ids of the fixed-size per-request state slots."""

    def take_one(self) -> int:
        try:
            return self.take(1)[0]
        except OutOfPages:
            raise OutOfSlots(f"all {self.num_pages} request slots are in use") from None
