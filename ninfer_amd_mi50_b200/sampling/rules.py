"""Penalties, biases and sets of allowed tokens of a step's rows, on the device.

The tokens of every request that a penalty looks at are kept in a log on the device; a step brings only those that the
log lacks (one a request while it decodes).  All index data of a step cross in one copy.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Hashable, List, Optional, Sequence

import numpy as np
import torch

from .. import kernels
from .params import SamplingParams


def mask_words(ids: Sequence[int], vocab: int) -> np.ndarray:
    """int32 words whose bit i % 32 of word i // 32 is set for the given ids."""
    on = np.zeros(((vocab + 31) // 32) * 32, dtype=bool)
    ids = np.asarray(list(ids), dtype=np.int64)
    if ids.size and not (0 <= ids.min() and ids.max() < vocab):
        raise ValueError(f"allowed tokens from {ids.min()} to {ids.max()} do not lie in [0, {vocab})")
    on[ids] = True
    return np.packbits(on, bitorder="little").view(np.int32)


@dataclass
class RuleRow:
    """One row of logits that has rules."""
    row: int
    params: SamplingParams
    tokens: Sequence[int]                  # the request's tokens so far, prompt and generated
    prompt_length: int
    key: Hashable                          # the request; None: of no request, its log is not kept
    allowed: Optional[Sequence[int]]       # the tokens that may follow; None: any


class TokenLogs:
    """Logs of tokens on the device, one a request."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.history: Optional[torch.Tensor] = None          # int32 [slots, capacity]
        self.slots: Dict[Hashable, int] = {}
        self.known: List[int] = []                           # tokens that a slot's log holds

    def forget(self, key: Hashable) -> None:
        self.slots.pop(key, None)

    def fit(self, slots: int, capacity: int) -> None:
        """Room for so many logs of so many tokens.  A larger tensor begins empty: the logs are sent again."""
        have = (0, 0) if self.history is None else tuple(self.history.shape)
        if have[0] >= slots and have[1] >= capacity:
            return
        shape = (max(slots, have[0], 8), (max(capacity, 2 * have[1], 1024) + 3) // 4 * 4)
        self.history = torch.zeros(shape, dtype=torch.int32, device=self.device)
        self.slots, self.known = {}, [0] * shape[0]

    def place(self, rows: Sequence[RuleRow]) -> List[int]:
        """The slot of each row's log; logs of requests that are not among them give way where there is no room."""
        self.fit(len(rows), max(len(r.tokens) for r in rows))
        here = {r.key for r in rows if r.key is not None}
        free = [s for s in range(len(self.known)) if s not in self.slots.values()]
        out = []
        for r in rows:
            slot = self.slots.get(r.key) if r.key is not None else None
            if slot is None:
                if not free:
                    old = next(k for k in self.slots if k not in here)
                    free.append(self.slots.pop(old))
                slot = free.pop()
                self.known[slot] = 0
                if r.key is not None:
                    self.slots[r.key] = slot
            out.append(slot)
        return out


def apply_rules(logits: torch.Tensor, rows: Sequence[RuleRow], logs: TokenLogs, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 [R, V] -> the same with the rules of the given rows; the other rows as they are."""
    R, V = logits.shape
    device = logits.device
    back = [r for r in rows if r.params.penalises]
    slots, lengths, starts = np.zeros(R, np.int32), np.zeros(R, np.int32), np.zeros(R, np.int32)
    penalties = np.tile(np.array([1.0, 0.0, 0.0], np.float32), (R, 1))
    tokens, held = np.zeros(0, np.int32), {}               # held: slots -> the tokens that their logs have after this
    placed = np.zeros((2, 0), np.int32)
    if back:
        new_tokens, new_slots, new_at = [], [], []
        for r, slot in zip(back, logs.place(back)):
            n, known = len(r.tokens), logs.known[slot]
            slots[r.row], lengths[r.row], starts[r.row] = slot, n, min(r.prompt_length, n)
            penalties[r.row] = r.params.repetition_penalty, r.params.frequency_penalty, r.params.presence_penalty
            if known > n:                                    # a log never shrinks: this is another list of tokens
                known = 0
            new_tokens += r.tokens[known:]
            new_slots += [slot] * (n - known)
            new_at += range(known, n)
            held[slot] = n
        tokens, placed = np.asarray(new_tokens, np.int32), np.asarray([new_slots, new_at], np.int32)
    else:
        logs.fit(1, 4)
    offsets, ids, values = np.zeros(R + 1, np.int32), [], []
    for r in sorted(rows, key=lambda r: r.row):
        bias = r.params.logit_bias or {}
        offsets[r.row + 1] = len(bias)
        ids += (int(t) for t in bias)
        values += bias.values()
    offsets = np.cumsum(offsets, dtype=np.int32)
    index, words = np.full(R, -1, np.int32), []
    for r in rows:
        if r.allowed is not None:
            index[r.row] = len(words)
            words.append(mask_words(r.allowed, V))
    pieces = [slots, lengths, starts, penalties.reshape(-1).view(np.int32), tokens, placed.reshape(-1), offsets, np.asarray(ids, np.int32),
              np.asarray(values, np.float32).view(np.int32), index, *words]
    host = torch.from_numpy(np.concatenate(pieces))
    sent = host.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else host
    slots_d, lengths_d, starts_d, pen_d, tok_d, placed_d, off_d, ids_d, val_d, index_d, words_d = sent.split(
        [len(p) for p in pieces[:10]] + [sum(len(w) for w in words)])
    if len(tokens):
        kernels.append_history(logs.history, placed_d[:len(tokens)], placed_d[len(tokens):], tok_d)
    for slot, n in held.items():             # (not before: a call that fails on the way has sent nothing)
        logs.known[slot] = n
    return kernels.adjust_logits(
        logits, logs.history, slots_d, lengths_d, starts_d, pen_d.view(torch.float32).view(R, 3),
        bias=(off_d, ids_d, val_d.view(torch.float32)) if ids else None,
        mask=(words_d.view(len(words), -1), index_d) if words else None, out=out)
