"""The plan of an attention step whose rows share the first keys of their contexts in groups.

A step of single-token rows falls into runs of rows; the rows of a run share their first ``keys`` keys, read through the block
table of the run's first row.  The plan cuts the step into items, each one workgroup a kv head (csrc/shared_attention.hip):
columns (query heads of rows) x keys, so that all items take about the same time and there are as many as compute units; the
short items of single rows come last and get a wave each.  Making one is host work, several times what the attention it plans takes (40 us for 4 rows,
81 for 32, 135 for 8 runs of 8, 247 for 256, the copy asked for but not waited for; three times that on slower hosts): it pays over a step's layers
and the steps that go on with it.
An item leaves a partial result for each of its columns; a row's partial results are its items in order of keys.
"""
from __future__ import annotations

from ctypes import addressof, c_long

import numpy as np
import torch

TILE = 64               # columns that a workgroup's four waves take with one tile of 16 each
BLOCK_KEYS = 32
LEAST_KEYS = 64         # of a cut: an item's start and its partial result cost about as much
START = 500             # what a workgroup's start and end cost, in keys of an item of up to 16 columns
LEAST_WIDE_KEYS = 192   # the same of items of more than 64 columns in bfloat16, whose partial results are the larger (32 rows behind 2,000
                        # keys in such items: cuts of 64 keys 22 us, of 128 18.7, of 192 17.1, of 256 18.8; fourteen drawn shapes whose cuts
                        # this moves, 5 to 146 rows behind 1,000 to 11,600 keys, in geometric mean of 64 to 192 18.5, of 256 17.4, of 320 17.7)


def _sharers(head_dim: int, float32: bool) -> int:
    """How many of a workgroup's waves share the keys of an item of up to 16 columns, or have such items of their own; 0: one wave takes all its keys."""
    row_bytes = head_dim * (4 if float32 else 2)
    return 0 if row_bytes % 64 else 4 if row_bytes <= 256 else 2


class SharedPrefixPlan:
    """Who shares what in a step of single-token rows.  ``groups``: (rows, keys) of every run of rows, in order; ``contexts``: the
    most keys each row has while the plan is used (its position + 1, or more: a plan holds for as many steps as its rows and
    shared keys stay and their contexts suffice; keys behind them are not seen).  Made once a step, or once for many, and used by every
    layer of it, in captured graphs as well as long as it is kept, but not made while a stream records.  ``share``: whether shared keys are read once for all
    (True), by every row for itself (False), or what is faster (None)."""

    def __init__(self, groups, contexts, num_q_heads: int, num_kv_heads: int, head_dim: int, device, units: int = 256,
                 float32: bool = False, share: bool | None = None):
        self.contexts = np.array(contexts, dtype=np.int64).reshape(-1)
        contexts = self.contexts.tolist()
        groups = [(int(n), int(k)) for n, k in groups]
        if num_kv_heads < 1 or num_q_heads < 1 or num_q_heads % num_kv_heads:
            raise ValueError(f"shared prefix: {num_q_heads} query heads are not a multiple of {num_kv_heads} kv heads")
        if any(n < 1 or k < 0 for n, k in groups) or sum(n for n, _ in groups) != len(contexts):
            raise ValueError(f"shared prefix: runs of rows {groups[:8]} for {len(contexts)} rows")
        self.max_context = max(contexts, default=0)
        if min(contexts, default=0) < 0 or self.max_context > 0x7FFFFF00:
            raise ValueError("shared prefix: contexts are numbers of keys, 0 or more")
        first = 0
        for n, k in groups:
            if min(contexts[first:first + n]) < k:
                raise ValueError(f"shared prefix: rows {first} to {first + n - 1} share {k} keys, and one of them has fewer")
            first += n
        self.num_rows, self.num_q_heads, self.num_kv_heads, self.head_dim = len(contexts), int(num_q_heads), int(num_kv_heads), int(head_dim)
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
        # What a key of an item costs, in keys of an item of up to 16 columns, whose waves share out the keys: measured, us for 64 keys in
        # bfloat16 0.4, of up to 64 columns 0.9, of 128 columns 1.3 (head size 128); the products of float32 weigh more.
        def weigh(column_tiles):
            wide = TILE * column_tiles
            tiles = [-(-w[1] // wide) for w in work]
            cost = [1 if w[1] <= 16 else (4 if float32 else 2) if min(w[1], wide) <= TILE else 3 for w in work]
            return wide, tiles, cost, sum(t * c * (w[3] - w[2]) for w, t, c in zip(work, tiles, cost)) * num_kv_heads

        # 128 columns a workgroup cost less than twice 64, but where there is little to do 64 leave the keys in fewer pieces to join (32 rows of 32 / 8
        # heads behind 2,000 keys, 190 keys a unit by these weights, 17.8 us and 19.2; 172 of 8 / 2 behind some 3,200, 450, 20.3 and 22.7; 2 times 107
        # of 32 / 4 behind some 800, 530, 19.7 and 18.2; 126 of 8 / 2 behind 16,712, 1,570, 26.9 and 23.5).
        self.column_tiles = 2 if max((w[1] for w in work), default=1) > TILE and head_dim <= 128 and not float32 else 1
        wide, tiles, cost, total = weigh(self.column_tiles)
        if self.column_tiles == 2 and total <= 600 * units:
            self.column_tiles = 1
            wide, tiles, cost, total = weigh(1)
        # One compute unit's share.  Items of half of it balance better and leave twice the partial results: over fifteen shapes in
        # geometric mean 35.3 us, 33.2 at two thirds, 31.9 at this, 33.9 at four thirds.  But two workgroups on a unit do 1.35 times what one does, which
        # long items are worth cutting for (two thirds: 256 rows behind 8,192 keys 118 -> 109 us, 77 of 56 / 7 heads of 32 behind 20,855 63 -> 53).
        most = -(-total // units)
        if most > 3000:
            most = -(-2 * most // 3)

        # Rows whose own keys are few next to a compute unit's share get a wave each: fewer workgroups, and nothing to join among the waves.  (236
        # rows of 48 / 6 heads of 64 behind 2,466 keys with 1 to 75 of their own 40.4 -> 37.8 us, 248 rows of 21 / 7 of 256 behind some 770 with
        # 1 to 63 79 -> 53; the 256 rows below 131 -> 116; 220 rows of 15 / 5 of 128 with 200 to 220 keys, whole, 20 -> 15, with 800 39 -> 43.)  Of
        # more workgroups than there is room for at once, the rows with up to 448 keys at any rate.
        sharers = _sharers(head_dim, float32) if G <= 16 else 0
        share_with_starts = sum(t * (c * (w[3] - w[2]) + START) for w, t, c in zip(work, tiles, cost)) * num_kv_heads / units
        few = (share_with_starts - START) / (2 * sharers) if sharers else 0
        if sharers and sum(w[1] == G for w in work) * num_kv_heads > 2 * units:
            few = max(few, 224 if float32 and sharers < 4 else 448)

        def cut(most):
            parts = [0] * self.num_rows
            items, several, solo = [], [], []
            for (row, columns, begin, end), t, c in zip(work, tiles, cost):
                least = LEAST_WIDE_KEYS if c == 3 else LEAST_KEYS
                pieces = 1 if whole and share is None else -(-(end - begin) // max(least, -(-most // (c * BLOCK_KEYS)) * BLOCK_KEYS))
                size = -(-(-(-(end - begin) // pieces)) // BLOCK_KEYS) * BLOCK_KEYS
                rows, at, part = columns // G, begin, parts[row]
                if rows == 1 and pieces == 1 and end - begin <= few:
                    solo.append((row, columns, 0, begin, end, part, 0, 0))
                    parts[row] = part + 1
                    continue
                while at < end:
                    # cuts lie on whole blocks of the cache, so that no block is read twice
                    to = end if end - at <= size else (at + size) // BLOCK_KEYS * BLOCK_KEYS
                    (several if rows > 1 else items).extend([(row, columns, i * wide, at, to, part, 0, 0) for i in range(t)])
                    part += 1
                    at = to
                parts[row:row + rows] = [part] * rows
            return parts, several, items, solo

        parts, several, items, solo = cut(most)
        # In float32 a few workgroups more than units cost almost a second round of them (24 rows of 32 / 4 heads of 64: 288 workgroups 16.6 us, 240 14.3;
        # sixteen drawn shapes of heads of 16 to 256 that this cuts otherwise, in geometric mean 20.6 and 19.3, eleven of them faster, five up to 16 % slower).
        groups = (len(several) + len(items) + -(-len(solo) // max(1, sharers))) * num_kv_heads
        if float32 and units < groups <= 1.25 * units:
            parts, several, items, solo = cut(most * 4 // 3)
        # the longest first: items of many columns take several times what those of one row do (256 rows behind 8,192 keys: the two kinds
        # spread among one another 256 us, these first 182)
        items = several + items
        self.whole_items = len(items)               # of a workgroup each; those of a wave each come after them, waves of like length side by side
        items += sorted(solo, key=lambda i: i[3] - i[4])
        self.num_items = len(items)
        starts = np.zeros(self.num_rows + 1, dtype=np.int32)
        np.cumsum(parts, out=starts[1:])
        self.num_parts = int(starts[-1])
        most_parts = max(parts, default=1)
        self.most_parts = 1 if most_parts == min(parts, default=1) == 1 else max(2, most_parts)      # 1: every row has one, nothing to join
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
        self._numbers = (c_long * 13)(*self.addresses, self.num_items, self.whole_items, self.column_tiles, self.most_parts, self.num_parts, self.num_rows,
                                      self.num_q_heads, self.num_kv_heads, self.head_dim, self.max_context, data.get_device())
        self.numbers = addressof(self._numbers)     # the same for csrc/direct_calls.hip

    def __deepcopy__(self, memo):
        return self                                 # nothing of a plan changes, and the addresses are of its own memory

    def __reduce__(self):
        raise TypeError("a plan is addresses of this process's memory")

    def exceeded_by(self, step) -> bool:
        """Whether a row of the step has more keys than it was planned for, as far as the host knows them."""
        ends = step.host.get("row_context") if step.host else None
        return ends is not None and bool((ends > self.contexts).any())

    def used_on(self, stream: int) -> None:
        """The current stream, ``stream`` by handle, is about to read the plan: another than its own waits for it and keeps its memory."""
        if stream != self.stream and self.ready is not None and not torch.cuda.is_current_stream_capturing():
            here = torch.cuda.current_stream(self._data.device)
            here.wait_event(self.ready)
            self._data.record_stream(here)

    def _worth_it(self, G: int, units: int, float32: bool) -> bool:
        """Whether contexts are cut and shared keys read once, or every row's whole context is left to one workgroup or wave a kv head, with no
        partial results and no second launch: as long as that takes no longer.  Measured, us, whole / shared by (rows x kv heads) / 256.
          bfloat16, heads of 64:   0.1: 700 keys 8 / 8, 1,500 keys 11 / 8;   0.5 to 2: 1,500 keys 11 to 14 / 13 to 14;   3: 800 keys 17 / 14;   4.3: 400 keys
          16 / 15;   8: 400 keys 15 / 19, 800 25 / 21
          of 128:    0.1 to 2: 1,000 keys 12 to 16 / 12 to 17;   3: 400 keys 15 / 17, 800 24 / 20;   4.3: 200 keys 15 / 18, 400 23 / 20;   8: 400 keys 21 / 27, 800
          35 / 27;   of 256:   0.1 to 2: 500 keys 16 to 24 / 14 to 22;   3: 200 keys 17 / 25, 400 24 / 26;   4.3: 100 keys 22 / 25, 200 32 / 27;   8: 200 keys 35 / 37
          float32, of 64:   0.1 to 1: 350 keys 10 / 9 to 12, 500 keys 13 / 10 to 14;   2: 200 keys 11 / 11, 400 16 / 13;   3: 100 keys 11 / 13, 200 16 / 14;   4.3: 100 keys
          16 / 14;   8: 100 keys 16 / 23, 200 24 / 27
          of 128:    0.1 to 1: 100 keys 11 / 13, 200 17 / 14;   2: 100 keys 16 / 16;   3: 30 keys 16 / 20, 100 25 / 18;   4.3: 30 keys 22 / 28;   8: 30 keys 31 / 40, 100 47 / 39
          of 256:    0.1 to 1: 100 keys 19 / 21, 200 30 / 21;   4: 100 keys 60 / 45
          one wave takes all keys, heads of 48 and 80:   0.1: 200 keys 8 / 7;   0.5 to 1: 350 keys 10 / 11 to 12, 500 12 to 13 / 11;   4: 200 keys 13 / 15, 350 17 / 15
          heads of 128 with 20 query heads each:   0.1: 350 keys 11 / 13, 500 14 / 12;   0.5: 500 keys 15 / 16, 700 18 / 17;   2: 700 keys 22 / 29;   float32:  0.1
          to 0.5: 100 keys 15 / 13 to 15;   2: 200 keys 35 / 36"""
        D, load = self.head_dim, self.num_rows * self.num_kv_heads / units
        sharers = _sharers(D, float32)
        if G > 16:
            most, rounds = (10000 // D * max(1, load), 1) if float32 else (min(640, 81920 // D), load / 3)
        elif not sharers:
            most, rounds = 420, load / 2
        elif float32:
            most, rounds = (28800 // D, max(min(load, 4), load / 4)) if sharers == 4 else (max(112, 17000 // D), max(min(load, 2.5), load / 4))
        else:
            most, rounds = min(1536 if load >= 0.5 else 900, 131072 // D), -(-load // 2) if load <= 6 else 0.3 * load
        return self.max_context * max(1, rounds) > most
