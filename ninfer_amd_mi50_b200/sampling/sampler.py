"""Choosing the next token from a row of logits.

The reference samples on the host from a copy of the logits (``sample_logits``,
src/runtime/engine.cpp:18-82): repetition penalty -> greedy if temperature <= 0 -> divide
by the temperature -> top-k -> softmax -> top-p -> inverse-CDF draw.  `Sampler` does the same
with device kernels; `sample_reference` is the host restatement used as the kernels' twin
and by ``Ninfer.sample`` when it is handed host logits.

Random draws are counter-based: the uniform number for a request's n-th new token depends
on (seed, n) only, so preempting a request and recomputing it later does not change what it
generates.  (The reference seeds a fresh Mersenne twister with ``seed + step`` per draw,
engine.cpp:166-169; the idea is the same, the generator is not.)
"""

from __future__ import annotations

import ctypes
import math
from collections import Counter
from typing import Hashable, List, Optional, Sequence

import torch

from .. import kernels
from .params import SamplingParams
from .rules import RuleRow, TokenLogs, apply_rules

_MASK = (1 << 64) - 1


def uniform_draw(seed: int, counter: int) -> float:
    """A float32-exact uniform number in [0, 1) from (seed, counter): splitmix64 mixing."""
    z = (seed * 0x9E3779B97F4A7C15 + (counter + 1) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK
    z ^= z >> 31
    return (z >> 40) / float(1 << 24)


def float32(v: float) -> float:
    """The number that the device computes with: an infinity for what float32 has no room for."""
    return ctypes.c_float(v).value


def check_allowed(ids: Sequence[int], vocab: int) -> None:
    for t in ids:
        if not 0 <= int(t) < vocab:
            raise ValueError(f"allowed token {t} outside [0, {vocab})")


def check_leaves(p: SamplingParams, ids: Sequence[int]) -> None:
    if not p.leaves(ids):
        raise ValueError("the allowed tokens and biases of -inf leave no token to draw")


def check_rules(p: SamplingParams, vocab: int) -> None:
    """Raises ValueError for penalties, biases or allowed tokens that make no sense."""
    if p.has_rules and not float32(p.repetition_penalty) > 0:
        raise ValueError("repetition_penalty must be positive")
    for what in ("frequency_penalty", "presence_penalty"):
        if not math.isfinite(float32(getattr(p, what))):
            raise ValueError(f"{what}={getattr(p, what)} must be finite")
    for t, v in (p.logit_bias or {}).items():
        if not 0 <= int(t) < vocab:
            raise ValueError(f"logit_bias names token {t} outside [0, {vocab})")
        if float(v) != -math.inf and not math.isfinite(float32(v)):
            raise ValueError(f"logit_bias of token {t} is {v}: finite, or -inf for a token that is never drawn")
    if p.allowed_tokens is not None and not callable(p.allowed_tokens):
        if len(p.allowed_tokens) == 0:
            raise ValueError("allowed_tokens allows nothing")
        check_allowed(p.allowed_tokens, vocab)
    if p.logit_bias:
        if len({int(t) for t in p.logit_bias}) < len(p.logit_bias):
            raise ValueError("logit_bias names a token twice")
        check_leaves(p, range(vocab) if p.allowed_tokens is None or callable(p.allowed_tokens) else p.allowed_tokens)


def check_params(p: SamplingParams, vocab: int) -> None:
    check_rules(p, vocab)
    check_draw(p, vocab)


def check_draw(p: SamplingParams, vocab: int) -> None:
    """Raises ValueError for limits of a draw that the device sampler does not take."""
    if p.greedy:
        return
    k = min(max(p.top_k, 1), vocab)
    if k > kernels.SAMPLE_MAX_TOP_K and not (k >= vocab and p.top_p >= 1.0):
        raise ValueError(
            f"top_k={p.top_k} is above {kernels.SAMPLE_MAX_TOP_K}; the device sampler takes a "
            f"larger top_k only as 'no limit' (top_k >= vocab) together with top_p >= 1")
    if p.repetition_penalty <= 0:
        raise ValueError("repetition_penalty must be positive")


def sample_reference(logits: Sequence[float], p: SamplingParams, recent: Sequence[int] = (),
                     draw: float = 0.0, prompt_length: int = 0) -> int:
    """Host twin: same policy, same tie rules, same draw.  `recent[prompt_length:]` are the generated ids."""
    l = torch.as_tensor(logits, dtype=torch.float32).clone()
    V = l.numel()
    if p.repetition_penalty != 1.0:
        for tok in recent:
            if 0 <= tok < V:
                l[tok] = l[tok] / p.repetition_penalty if l[tok] > 0 else l[tok] * p.repetition_penalty
    if p.has_rules:
        generated = list(recent[prompt_length:])
        for tok, n in Counter(generated).items():
            if 0 <= tok < V:
                l[tok] = l[tok] - n * p.frequency_penalty - p.presence_penalty
        for tok, v in (p.logit_bias or {}).items():
            l[int(tok)] += v
        allowed = p.allowed(generated)
        if allowed is not None:
            allowed = list(allowed)
            check_leaves(p, allowed)
            left_out = torch.ones(V, dtype=torch.bool)
            left_out[torch.as_tensor(allowed, dtype=torch.long)] = False
            l[left_out] = -math.inf
    if p.greedy:
        return int(torch.argmax(l))          # first maximum
    l = l * torch.tensor(1.0 / p.temperature, dtype=torch.float32)
    k = min(max(p.top_k, 1), V)
    if k >= V and p.top_p >= 1.0:
        e = torch.exp(l - l.max())
        cum = torch.cumsum(e, 0)
        # (a token of probability 0 is never drawn, here and below)
        hit = torch.nonzero((cum >= draw * e.sum()) & (e > 0))
        some = torch.nonzero(e > 0)
        return int(hit[0]) if len(hit) else int(some[-1]) if len(some) else V - 1
    order = sorted(range(V), key=lambda i: (-float(l[i]), i))[:k]
    vals = l[order]
    prob = torch.exp(vals - vals[0])
    prob = prob / prob.sum()
    keep = k
    if p.top_p < 1.0:
        cum = 0.0
        for i in range(k):
            cum += float(prob[i])
            if cum >= p.top_p:
                keep = i + 1
                break
    prob = prob[:keep] / prob[:keep].sum()
    cum, pick = 0.0, order[keep - 1]
    for i in range(keep):
        cum += float(prob[i])
        if prob[i] > 0:
            pick = order[i]
            if draw <= cum:
                break
    return pick


class Sampler:
    """Device sampling for a batch of rows with per-row parameters."""

    def __init__(self, vocab_size: int, device):
        self.vocab_size, self.device = vocab_size, torch.device(device)
        self.logs = TokenLogs(self.device)

    def forget(self, key: Hashable) -> None:
        """A request is done: its log of tokens may be given to another."""
        self.logs.forget(key)

    def sample(self, logits: torch.Tensor, params: Sequence[SamplingParams],
               recent: Optional[Sequence[Sequence[int]]] = None,
               counters: Optional[Sequence[int]] = None, prompt_lengths: Optional[Sequence[int]] = None,
               keys: Optional[Sequence[Hashable]] = None,
               allowed: Optional[Sequence[Optional[Sequence[int]]]] = None) -> torch.Tensor:
        """logits float32 [R, V] on the device -> int32 [R] on the device.

        `recent[r]` are the ids the penalties look at (prompt and generated), of which the first
        `prompt_lengths[r]` are the prompt's (0 if left out);
        `counters[r]` is the index of the token being drawn, the RNG counter; `keys[r]` names the request whose tokens
        these are, so that only new ones are sent; `allowed[r]` is what `params[r].allowed` says of the generated ids, where
        the caller has asked already."""
        R = logits.shape[0]
        if R == 0:
            return torch.empty((0,), dtype=torch.int32, device=self.device)
        dev = self.device
        # repetition penalty on a copy (the caller may still want the raw logits)
        rule_rows = [r for r in range(R) if params[r].has_rules]
        pen_rows = [r for r in range(R) if params[r].repetition_penalty != 1.0 and recent and recent[r] and not params[r].has_rules]
        own = bool(pen_rows)
        if pen_rows:
            logits = logits.clone()
            ids, counts, row_of = [], [], []
            for r in pen_rows:
                for tok, c in Counter(int(t) for t in recent[r]).items():
                    ids.append(tok); counts.append(c); row_of.append(r)
            mk = lambda v, dt: torch.tensor(v, dtype=dt).to(dev)
            pen = mk([p.repetition_penalty for p in params], torch.float32)
            kernels.repetition_penalty(logits, mk(ids, torch.int32), mk(counts, torch.int32),
                                       mk(row_of, torch.int32), pen)
        if rule_rows:
            rows = []
            for r in rule_rows:
                tokens = list(recent[r]) if recent else []
                prompt = prompt_lengths[r] if prompt_lengths else 0
                if allowed is not None:
                    ids = allowed[r]
                else:
                    ids = params[r].allowed(tokens[prompt:])
                    if ids is not None:
                        ids = list(ids) if callable(params[r].allowed_tokens) else ids
                        check_leaves(params[r], ids)
                rows.append(RuleRow(r, params[r], tokens, prompt, keys[r] if keys else None, ids))
            logits = apply_rules(logits, rows, self.logs, out=logits if own else None)
        if all(p.greedy for p in params):
            return kernels.argmax_rows(logits)
        out = kernels.argmax_rows(logits)
        rows = [r for r in range(R) if not params[r].greedy]
        for r in rows:
            (check_params if params[r].has_rules else check_draw)(params[r], self.vocab_size)
        sel = torch.tensor(rows, dtype=torch.long, device=dev)
        sub = logits.index_select(0, sel) if len(rows) < R else logits
        temp = torch.tensor([params[r].temperature for r in rows], dtype=torch.float32).to(dev)
        topk = torch.tensor([params[r].top_k for r in rows], dtype=torch.int32).to(dev)
        topp = torch.tensor([params[r].top_p for r in rows], dtype=torch.float32).to(dev)
        draws = torch.tensor([uniform_draw(params[r].seed, counters[r] if counters else 0) for r in rows],
                             dtype=torch.float32).to(dev)
        picked = kernels.sample_rows(sub.contiguous(), temp, topk, topp, draws)
        if len(rows) == R:
            return picked
        out.index_copy_(0, sel, picked)
        return out
