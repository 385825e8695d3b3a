"""Free lists of page ids and of state slots.

Page 0 (and slot 0) is scratch: never handed out; padded rows of a captured
decode step write there (inference_engine/block_manager.py:14-19).  Ids are
taken from the left and given back on the right, so a freed page is reused
after the ones freed before it (inference_engine/block_manager.py:39,43).  A
page that several requests read (a shared first part) is free once all of them
have given it back.
"""
from __future__ import annotations

from collections import deque


class CacheAccountingError(RuntimeError):
    """A page or slot was given back twice, was never taken, or is scratch."""


class IdPool:
    def __init__(self, count: int, reserved: int = 1, what: str = "page"):
        if count <= reserved:
            raise ValueError(f"need more than {reserved} {what}s, got {count}")
        self.count = count
        self.reserved = reserved
        self.what = what
        self.free = deque(range(reserved, count))
        self._held = [0] * count            # holders of each id
        self.low_water = len(self.free)

    @property
    def num_free(self) -> int:
        return len(self.free)

    @property
    def num_usable(self) -> int:
        return self.count - self.reserved

    def take(self, n: int) -> list[int] | None:
        if n > len(self.free):
            return None
        ids = [self.free.popleft() for _ in range(n)]
        for i in ids:
            self._held[i] = 1
        self.low_water = min(self.low_water, len(self.free))
        return ids

    def share(self, ids) -> None:
        """One more holder of ids that are held."""
        ids = list(ids)
        for i in ids:
            if not self.reserved <= i < self.count or not self._held[i]:
                raise CacheAccountingError(f"{self.what} {i} shared but not held")
        for i in ids:
            self._held[i] += 1

    def holders(self, i: int) -> int:
        return self._held[i]

    def give_back(self, ids) -> list[int]:
        """Those of the ids that nobody holds any more are free again, and returned."""
        freed = []
        for i in ids:
            if not self.reserved <= i < self.count:
                raise CacheAccountingError(f"{self.what} {i} is scratch or out of range")
            if not self._held[i]:
                raise CacheAccountingError(f"{self.what} {i} given back but not held")
            self._held[i] -= 1
            if not self._held[i]:
                self.free.append(i)
                freed.append(i)
        return freed

    def held(self) -> set[int]:
        return {i for i, h in enumerate(self._held) if h}
