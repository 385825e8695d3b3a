"""The plan of an attention step whose rows share the first keys of their contexts in groups.

A step of single-token rows falls into runs of rows; the rows of a run share their first ``keys`` keys, read through the block
table of the run's first row.  The plan cuts the step into items, each one workgroup a kv head (csrc/shared_attention.hip):
columns (query heads of rows) x keys, so that all items take about the same time and there are enough of them for
the GPU.  An item leaves a partial result for each of its columns; a row's partial results are its items in order of keys.
"""
from __future__ import annotations

import numpy as np
import torch

TILE = 64               # columns that a workgroup's four waves take with one tile of 16 each
BLOCK_KEYS = 32


class SharedPrefixPlan:
    """Who shares what in a step of single-token rows.  ``groups``: (rows, keys) of every run of rows, in order; ``contexts``: the
    most keys each row has while the plan is used (its position + 1, or more: a plan holds for as many steps as its rows and
    shared keys stay and their contexts suffice).  Made once a step, or once for many, and used by every layer of it."""

    def __init__(self, groups, contexts, num_q_heads: int, num_kv_heads: int, head_dim: int, device, units: int = 256, least_keys: int = 64, per_unit: float = 1):
        contexts = [int(c) for c in contexts]
        groups = [(int(n), int(k)) for n, k in groups]
        if num_kv_heads < 1 or num_q_heads % num_kv_heads:
            raise ValueError(f"shared prefix: {num_q_heads} query heads are not a multiple of {num_kv_heads} kv heads")
        if any(n < 1 or k < 0 for n, k in groups) or sum(n for n, _ in groups) != len(contexts):
            raise ValueError(f"shared prefix: runs of rows {groups[:8]} for {len(contexts)} rows")
        if any(c < 0 or c > 0x7FFFFF00 for c in contexts):
            raise ValueError("shared prefix: contexts are numbers of keys, 0 or more")
        self.num_rows, self.num_q_heads, self.num_kv_heads, self.head_dim = len(contexts), int(num_q_heads), int(num_kv_heads), int(head_dim)
        self.contexts = np.asarray(contexts, dtype=np.int64)
        self.max_context = max(contexts, default=0)
        G = num_q_heads // num_kv_heads
        first, work = 0, []                         # (first row, columns, first key, keys) of what is to be cut
        for n, k in groups:
            if any(c < k for c in contexts[first:first + n]):
                raise ValueError(f"shared prefix: rows {first} to {first + n - 1} share {k} keys, and one of them has fewer")
            if n == 1:
                k = 0                               # nobody to share with
            elif k:
                work.append((first, n * G, 0, k))
            for r in range(first, first + n):
                if contexts[r] > k:
                    work.append((r, G, k, contexts[r]))
            first += n
        widest = max((w[1] for w in work), default=1)
        self.column_tiles = 2 if widest > TILE and head_dim <= 128 else 1
        wide = TILE * self.column_tiles
        tiles = [-(-w[1] // wide) for w in work]
        total = sum(t * (w[3] - w[2]) for w, t in zip(work, tiles)) * num_kv_heads
        # keys an item: two items a compute unit, and no less than 64 (an item's start and its partial result cost about as much)
        most = max(least_keys, -(-total // int(per_unit * units) // BLOCK_KEYS) * BLOCK_KEYS)
        parts = np.zeros(self.num_rows, dtype=np.int64)
        items, several = [], []
        for (row, columns, begin, end), t in zip(work, tiles):
            pieces = -(-(end - begin) // most)
            size = -(-(-(-(end - begin) // pieces)) // BLOCK_KEYS) * BLOCK_KEYS
            rows = columns // G
            at = begin
            while at < end:
                # cuts lie on whole blocks of the cache, so that no block is read twice
                to = end if end - at <= size else (at + size) // BLOCK_KEYS * BLOCK_KEYS
                (several if rows > 1 else items).extend((row, columns, c * wide, at, to, int(parts[row]), 0, 0) for c in range(t))
                parts[row:row + rows] += 1
                at = to
        # the longest first: items of many columns take several times what those of one row do (256 rows behind 8,192 keys: the two kinds
        # spread among one another 256 us, these first 182)
        items = several + items
        self.num_items = len(items)
        starts = np.zeros(self.num_rows + 1, dtype=np.int32)
        np.cumsum(parts, out=starts[1:])
        self.num_parts = int(starts[-1])
        self.most_parts = 1 if (parts == 1).all() else max(2, int(parts.max()))      # 1: every row has one, nothing to join
        self.join = self.most_parts != 1
        packed = np.concatenate([np.asarray(items, dtype=np.int32).reshape(-1), starts])
        data = torch.from_numpy(packed)
        if torch.device(device).type == "cuda":
            data = data.pin_memory().to(device, non_blocking=True)
        self._data = data
        self.items, self.row_parts = data[:8 * len(items)], data[8 * len(items):]
        self.addresses = self.items.data_ptr(), self.row_parts.data_ptr()
