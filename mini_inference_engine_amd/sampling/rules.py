"""From requests' options to the LogitRules of a step: penalties for tokens already there, biases, and masks of what may come.

The texts that penalties look at are on the device already (ModelRunner.token_history, written as the steps' tokens run), so a token
that the step before chose and the host has not seen counts like any other.  Everything else is a few numbers a row, packed into
one array and sent with one copy from a pinned buffer.
"""
from __future__ import annotations

import numpy as np
import torch

from ..kernels.api import LogitRules


def mask_words(allowed, vocab_size: int) -> np.ndarray:
    """Token ids as bits: token v is bit v % 32 of word v // 32."""
    words = (vocab_size + 31) // 32
    ids = np.fromiter((int(t) for t in allowed), dtype=np.int64)
    if ids.size and (ids.min() < 0 or ids.max() >= vocab_size):
        raise ValueError(f"allowed tokens outside the vocabulary of {vocab_size}: {ids[(ids < 0) | (ids >= vocab_size)][:5].tolist()}")
    bits = np.zeros(words * 32, dtype=np.uint8)
    bits[ids] = 1
    return np.packbits(bits, bitorder="little").view(np.int32)


class RuleInputs:
    """Makes the LogitRules of a step's rows.  Two pinned buffers take turns: the copy out of one may still be under way while the
    next step's rules are written to the other."""

    def __init__(self, device, vocab_size: int, stop_token_ids=()):
        self.device, self.vocab_size = torch.device(device), int(vocab_size)
        self.stop_token_ids = sorted(stop_token_ids)
        self._mirrors, self._copied, self._turn = [None, None], [None, None], 0
        self.asked = None               # the request whose allowed_tokens was last asked, until its answer is taken

    def _mirror(self, n: int) -> torch.Tensor:
        self._turn ^= 1
        if self._copied[self._turn] is not None:
            self._copied[self._turn].synchronize()
        m = self._mirrors[self._turn]
        if m is None or m.numel() < n:
            m = self._mirrors[self._turn] = torch.empty(max(n, 4096), dtype=torch.int32, pin_memory=self.device.type == "cuda")
        return m

    def make(self, seqs, lengths, history) -> LogitRules | None:
        """The rules of rows whose tokens are chosen for ``seqs``, ``lengths`` tokens of each known by then; None if nobody has any."""
        params = [s.params for s in seqs]
        self.asked = None
        if not any(p.has_rules for p in params):
            return None
        pieces, where = [], {}

        def put(name, numbers, dtype=np.int32):
            where[name] = (sum(len(p) for p in pieces), len(numbers))
            pieces.append(np.asarray(numbers, dtype=dtype).view(np.int32))

        if any(p.has_penalties for p in params):
            if history is None:
                raise ValueError("penalties look at the requests' texts, which nobody keeps (ModelRunner.keep_token_history)")
            put("slots", [s.cache.state_slot for s in seqs])
            put("lengths", lengths)
            put("prompt_lengths", [s.prompt_len for s in seqs])
            for name in ("repetition", "presence", "frequency"):
                put(name, [getattr(p, name + "_penalty") for p in params], np.float32)
        if any(p.logit_bias for p in params):
            lists = [p.logit_bias or {} for p in params]
            put("bias_starts", np.cumsum([0] + [len(b) for b in lists]))
            put("bias_tokens", [t for b in lists for t in b])
            put("bias_values", [v for b in lists for v in b.values()], np.float32)
        masks = {}                      # row -> words
        for i, s in enumerate(seqs):
            if s.params.allowed_tokens is None:
                continue
            self.asked = s
            allowed = s.params.allowed_tokens(list(s.output_ids))
            if allowed is None:
                continue
            words = mask_words(allowed, self.vocab_size)
            if not words.any():         # nothing can follow: the request may only end
                if not self.stop_token_ids:
                    raise ValueError(f"request {s.seq_id}: no token is allowed after {s.num_output_tokens}, and the model has no stop token")
                words = mask_words(self.stop_token_ids, self.vocab_size)
            masks[i] = words
        self.asked = None
        if masks:
            at = {i: j for j, i in enumerate(masks)}
            put("mask_rows", [at.get(i, -1) for i in range(len(seqs))])
            put("masks", np.concatenate(list(masks.values())))
        if not pieces:
            return None
        packed = np.concatenate(pieces)
        host = self._mirror(len(packed))
        host.numpy()[:len(packed)] = packed
        if self.device.type == "cuda":
            dev = torch.empty(len(packed), dtype=torch.int32, device=self.device)
            dev.copy_(host[:len(packed)], non_blocking=True)
            if self._copied[self._turn] is None:
                self._copied[self._turn] = torch.cuda.Event()
            self._copied[self._turn].record()
        else:
            dev = host[:len(packed)].clone()
        rules = LogitRules(history=history if "slots" in where else None)
        if rules.history is not None:
            rules.readers = torch.tensor([i for i, p in enumerate(params) if p.has_penalties])
        for name, (a, n) in where.items():
            t = dev[a:a + n]
            if name in ("repetition", "presence", "frequency", "bias_values"):
                t = t.view(torch.float32)
            setattr(rules, name, t.view(len(masks), -1) if name == "masks" else t)
        return rules
