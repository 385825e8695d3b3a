"""The plan of an attention step whose rows share the first keys of their contexts in groups.

A step of single-token rows falls into runs of rows; the rows of a run share their first ``keys`` keys, read through the block
table of the run's first row.  The plan cuts the step into items, each one workgroup a kv head (csrc/shared_attention.hip):
columns (query heads of rows) x keys, so that all items take about the same time and there are as many as compute units.
An item leaves a partial result for each of its columns; a row's partial results are its items in order of keys.
"""
from __future__ import annotations

import numpy as np
import torch

TILE = 64               # columns that a workgroup's four waves take with one tile of 16 each
BLOCK_KEYS = 32
LEAST_KEYS = 64         # of a cut: an item's start and its partial result cost about as much
LEAST_WIDE_KEYS = 192   # the same of items of more than 64 columns in bfloat16, whose partial results are the larger (32 rows behind 2,000
                        # keys: cuts of 64 keys 22 us, of 128 18.7, of 192 17.1, of 256 18.8)


class SharedPrefixPlan:
    """Who shares what in a step of single-token rows.  ``groups``: (rows, keys) of every run of rows, in order; ``contexts``: the
    most keys each row has while the plan is used (its position + 1, or more: a plan holds for as many steps as its rows and
    shared keys stay and their contexts suffice; keys behind them are not seen).  Made once a step, or once for many, and used by every
    layer of it, in captured graphs as well as long as it is kept, but not made while a stream records.  ``share``: whether shared keys are read once for all
    (True), by every row for itself (False), or what is faster (None)."""

    def __init__(self, groups, contexts, num_q_heads: int, num_kv_heads: int, head_dim: int, device, units: int = 256,
                 float32: bool = False, share: bool | None = None):
        contexts = [int(c) for c in contexts]
        groups = [(int(n), int(k)) for n, k in groups]
        if num_kv_heads < 1 or num_q_heads < 1 or num_q_heads % num_kv_heads:
            raise ValueError(f"shared prefix: {num_q_heads} query heads are not a multiple of {num_kv_heads} kv heads")
        if any(n < 1 or k < 0 for n, k in groups) or sum(n for n, _ in groups) != len(contexts):
            raise ValueError(f"shared prefix: runs of rows {groups[:8]} for {len(contexts)} rows")
        if any(c < 0 or c > 0x7FFFFF00 for c in contexts):
            raise ValueError("shared prefix: contexts are numbers of keys, 0 or more")
        first = 0
        for n, k in groups:
            if any(c < k for c in contexts[first:first + n]):
                raise ValueError(f"shared prefix: rows {first} to {first + n - 1} share {k} keys, and one of them has fewer")
            first += n
        self.num_rows, self.num_q_heads, self.num_kv_heads, self.head_dim = len(contexts), int(num_q_heads), int(num_kv_heads), int(head_dim)
        self.contexts = np.asarray(contexts, dtype=np.int64)
        self.max_context = max(contexts, default=0)
        G = num_q_heads // num_kv_heads
        whole = not self._worth_it(G, units, float32) if share is None else not share
        if whole:
            groups = [(1, 0)] * self.num_rows

        first, work = 0, []                         # (first row, columns, first key, end) of what is to be cut
        for n, k in groups:
            k = 0 if n == 1 else k                  # a single row has nobody to share with
            if k:
                work.append((first, n * G, 0, k))
            work += [(r, G, k, contexts[r]) for r in range(first, first + n) if contexts[r] > k]
            first += n
        widest = max((w[1] for w in work), default=1)
        self.column_tiles = 2 if widest > TILE and head_dim <= 128 else 1
        wide = TILE * self.column_tiles
        tiles = [-(-w[1] // wide) for w in work]
        # What a key of an item costs, in keys of an item of up to 16 columns, whose waves share out the keys: measured, us for 64 keys in
        # bfloat16 0.4, of up to 64 columns 0.9, of 128 columns 1.3 (head size 128); the 32-bit products of float32 weigh more.
        wider = (4, 8) if float32 else (2, 3)
        cost = [1 if w[1] <= 16 else wider[min(w[1], wide) > TILE] for w in work]
        total = sum(t * c * (w[3] - w[2]) for w, t, c in zip(work, tiles, cost)) * num_kv_heads
        # One compute unit's share.  Items of half of it balance better and leave twice the partial results: over fifteen shapes in
        # geometric mean 35.3 us, 33.2 at two thirds, 31.9 at this, 33.9 at four thirds.
        most = -(-total // units)

        parts = np.zeros(self.num_rows, dtype=np.int64)
        items, several = [], []
        for (row, columns, begin, end), t, c in zip(work, tiles, cost):
            least = LEAST_WIDE_KEYS if c == wider[1] and not float32 else LEAST_KEYS
            pieces = 1 if whole and share is None else -(-(end - begin) // max(least, -(-most // (c * BLOCK_KEYS)) * BLOCK_KEYS))
            size = -(-(-(-(end - begin) // pieces)) // BLOCK_KEYS) * BLOCK_KEYS
            rows = columns // G
            at = begin
            while at < end:
                # cuts lie on whole blocks of the cache, so that no block is read twice
                to = end if end - at <= size else (at + size) // BLOCK_KEYS * BLOCK_KEYS
                (several if rows > 1 else items).extend((row, columns, i * wide, at, to, int(parts[row]), 0, 0) for i in range(t))
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
        self.stream = self.ready = None             # where the plan was sent from, and the event behind its copy
        if torch.device(device).type == "cuda":
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("shared prefix: a plan is made before a capture, not in it (a replay would send its host memory again)")
            stream = torch.cuda.current_stream(device)
            data = data.pin_memory().to(device, non_blocking=True)
            self.stream, self.ready = stream.cuda_stream, torch.cuda.Event()
            self.ready.record(stream)
        self._data = data
        self.items, self.row_parts = data[:8 * len(items)], data[8 * len(items):]
        self.addresses = self.items.data_ptr(), self.row_parts.data_ptr()

    def used_on(self, stream: int) -> None:
        """The current stream, ``stream`` by handle, is about to read the plan: another than its own waits for it and keeps its memory."""
        if stream != self.stream and self.ready is not None and not torch.cuda.is_current_stream_capturing():
            here = torch.cuda.current_stream(self._data.device)
            here.wait_event(self.ready)
            self._data.record_stream(here)

    def _worth_it(self, G: int, units: int, float32: bool) -> bool:
        """Whether contexts are cut and shared keys read once, or every row's whole context is left to one workgroup a kv head, with no partial
        results and no second launch: as long as that takes no longer than the second launch costs.  Measured, us a call one after another,
        whole / shared.  4 kv heads of 64: 4 to 64 rows of 500 keys 11.6 / 16.1, of 1,000 11.7 / 16.1, 256 rows (two rounds of workgroups) of 500
        17.5 / 23.4, of 1,000 21.6 / 25.9.  8 of 128: 4 to 64 rows of 500 keys 11.6 / 16.0, of 1,000 11.7 to 15.9 / 16.2 to 17.8, 256 rows of 200 28.8 /
        36.3, of 500 39.4 / 38.6.  float32, 4 of 64: 200 keys 11.5 / 16.1, 500 keys 13.0 / 16.2, 1,000 keys 18.8 / 16.1; 8 of 128: 200 keys 12.0 to
        23.7 / 15.9 to 28.3, 500 keys 21.3 to 41.0 / 15.8 to 32.1."""
        D, rounds = self.head_dim, -(-self.num_rows * self.num_kv_heads // (2 * units))
        if G > 16 or D % 32 or D * (4 if float32 else 2) > 512:
            most = 128                              # one wave of four computes: see csrc/shared_attention.hip
        else:
            most = min(512, 32768 // D) if float32 else min(1536, 131072 // D)
        return self.max_context * rounds > most
