"""Rows of logits with masks, and draws at both ends, for the tests of the sampler and of its host twin."""

import torch

DRAWS = (0.0, 1.0 - 2.0 ** -24)       # the smallest and the largest that `uniform_draw` gives


def masked_rows(rows, V, seed):
    """(logits float32 [rows, V], allowed bool [rows, V]): -inf where not allowed; the first and the last token are left out of
    most rows, between 1 and V - 2 tokens are allowed."""
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(rows, V, generator=g) * 3
    allowed = torch.zeros(rows, V, dtype=torch.bool)
    for r in range(rows):
        n = int(torch.randint(1, min(V - 1, 1 + 4 ** (r % 8 + 1)), (1,), generator=g))
        allowed[r, 1 + torch.randperm(V - 2, generator=g)[:n]] = True
        if r % 7 == 0:
            allowed[r, 0] = allowed[r, V - 1] = True
    logits[~allowed] = -float("inf")
    return logits, allowed
