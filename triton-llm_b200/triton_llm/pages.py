"""Host-side accounting of a paged KV cache's pages: taking, sharing, releasing
and compacting them (no counterpart in the reference, whose caches are
preallocated per sequence). The pages' contents live on the device
(``triton_llm.kernels.paged``); this is only who uses which.
"""

from __future__ import annotations

import heapq

import numpy as np


class PagePool:
    """``n_pages`` pages with the number of users of each. A page is given out
    with one user; sequences that share it add theirs, and it is free again
    when the last one releases it. The lowest free pages go first, which keeps
    the used ones together."""

    def __init__(self, n_pages: int):
        if n_pages < 0:
            raise ValueError(f"n_pages must be >= 0, got {n_pages}")
        self.n_pages = int(n_pages)
        self.users = np.zeros(self.n_pages, np.int32)
        self._free = list(range(self.n_pages))   # a heap

    @property
    def free(self) -> int:
        return len(self._free)

    @property
    def used(self) -> int:
        return self.n_pages - len(self._free)

    def take(self, n: int) -> np.ndarray:
        """n free pages, each with one user. Takes none if there are fewer."""
        if n < 0:
            raise ValueError(f"cannot take {n} pages")
        if n > len(self._free):
            raise RuntimeError(f"out of pages: {n} asked for, {len(self._free)} of "
                               f"{self.n_pages} free")
        pages = np.array([heapq.heappop(self._free) for _ in range(n)], np.int32)
        self.users[pages] = 1
        return pages

    def _check(self, pages):
        pages = np.asarray(pages, np.int64).reshape(-1)
        if ((pages < 0) | (pages >= self.n_pages)).any():
            raise ValueError(f"pages {pages.tolist()} are not all in [0, {self.n_pages})")
        if (self.users[pages] == 0).any():
            raise ValueError(f"pages {pages[self.users[pages] == 0].tolist()} are free")
        return pages

    def share(self, pages) -> None:
        """One more user for every page (as often as it is named)."""
        np.add.at(self.users, self._check(pages), 1)

    def release(self, pages) -> None:
        """One user less for every page; those without one are free again."""
        pages = self._check(pages)
        count = np.bincount(pages, minlength=self.n_pages)
        if (count > self.users).any():
            raise ValueError(f"pages {np.flatnonzero(count > self.users).tolist()} are "
                             "released more often than they are used")
        self.users -= count.astype(np.int32)
        for p in np.unique(pages):
            if self.users[p] == 0:
                heapq.heappush(self._free, int(p))

    def compact(self):
        """Moves the used pages to the front of the pool. Returns (src, dst,
        where): the page copies that this needs (no page is in both) and
        ``where[p]``, the new place of page p (p itself for the others)."""
        used = self.used
        src = np.flatnonzero(self.users[used:]) + used
        dst = np.flatnonzero(self.users[:used] == 0)
        where = np.arange(self.n_pages, dtype=np.int32)
        where[src] = dst
        self.users[dst] = self.users[src]
        self.users[src] = 0
        self._free = list(range(used, self.n_pages))
        return src.astype(np.int32), dst.astype(np.int32), where
