"""Sampling parameters, with the reference's names, meanings and defaults
(``SamplingParams``, src/runtime/engine.h:15-22; CLI flags src/apps/ninfer.cpp:55-76)."""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Dict, Optional, Sequence, Union


@dataclass
class SamplingParams:
    temperature: float = 0.7          # <= 0: greedy (first maximum)
    top_k: int = 50                   # clamped to [1, vocab]
    top_p: float = 0.95               # >= 1: no nucleus cut
    repetition_penalty: float = 1.0   # 1: off (the CLI's default is 1.05, as in the reference)
    seed: int = 0                     # 0: a fresh seed per request
    max_new_tokens: int = 512
    # what the reference does not have: penalties on what was generated (each occurrence, and once), values added to
    # single tokens' logits, and the tokens that may follow: a set, or a function from the generated ids to one (None: any
    # token; an answer that is empty, or all of whose tokens have a bias of -inf, ends the request)
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None
    allowed_tokens: Union[Sequence[int], Callable[[Sequence[int]], Optional[Sequence[int]]], None] = None

    @property
    def greedy(self) -> bool:
        return self.temperature <= 0.0

    @property
    def has_rules(self) -> bool:
        """Whether logits pass through more than the repetition penalty."""
        return (self.frequency_penalty != 0.0 or self.presence_penalty != 0.0 or bool(self.logit_bias)
                or self.allowed_tokens is not None)

    @property
    def penalises(self) -> bool:
        return self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0 or self.presence_penalty != 0.0

    @property
    def looks_back(self) -> bool:
        """Whether the next token depends on earlier ones by more than the model."""
        return self.penalises or callable(self.allowed_tokens)

    def allowed(self, generated: Sequence[int]) -> Optional[Sequence[int]]:
        """The tokens that may follow `generated`; None: any."""
        a = self.allowed_tokens
        return a(list(generated)) if callable(a) else a

    def leaves(self, ids: Sequence[int]) -> bool:
        """Whether a token of `ids` may be drawn: one without a bias of -inf."""
        never = {int(t) for t, v in (self.logit_bias or {}).items() if v == -math.inf}
        return any(int(t) not in never for t in ids)
