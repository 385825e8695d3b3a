"""Per-request sampling options, as the reference names them
(inference_engine/sampling.py:6-10), plus a seed and the rules a request's tokens are chosen
under (kernels.api.LogitRules says what each does to a logit, and in which order)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable


@dataclass
class SamplingParams:
    max_tokens: int = 128
    temperature: float = 0.0        # 0 = greedy
    ignore_eos: bool = False        # keep generating past the stop token
    seed: int | None = None         # noise stream of this request; None: derived from the engine's seed
    repetition_penalty: float = 1.0  # > 0; logits of tokens in prompt or output are divided (above 0) or multiplied by it
    presence_penalty: float = 0.0   # taken from the logits of tokens in the output
    frequency_penalty: float = 0.0  # the same, times how often they occur there
    logit_bias: dict | None = None  # token id -> what is added to its logit
    # Which tokens may come next: called with the output so far before each token, gives token ids, or None for all.  Where
    # nothing may come, the stop tokens may.  The engine then reads every token before it starts the next step, as long as such a
    # request is there, queued or running.  What it raises, LLMEngine.step raises (LLMEngine.failed_request, LLMEngine.abort).
    allowed_tokens: Callable | None = None

    def __post_init__(self):
        if self.max_tokens < 0:
            raise ValueError("max_tokens must be >= 0")
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0")
        if not (0 < self.repetition_penalty < math.inf):
            raise ValueError("repetition_penalty must be a number above 0")
        if not (math.isfinite(self.presence_penalty) and math.isfinite(self.frequency_penalty)):
            raise ValueError("presence_penalty and frequency_penalty must be finite")
        for token, value in (self.logit_bias or {}).items():
            if not isinstance(token, int) or math.isnan(value):
                raise ValueError(f"logit_bias: token id {token!r} with {value!r}")
        if self.allowed_tokens is not None and not callable(self.allowed_tokens):
            raise ValueError("allowed_tokens is called with the output so far; give a function")

    @property
    def has_penalties(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    @property
    def has_rules(self) -> bool:
        return self.has_penalties or bool(self.logit_bias) or self.allowed_tokens is not None
