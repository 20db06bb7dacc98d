"""Draws from rows with masks by the host twin: never a token of probability 0."""

import pytest
import torch

from draw_cases import DRAWS, masked_rows

from ninfer_amd_mi50_b200.sampling import SamplingParams, sample_reference

POLICIES = [(500, 1.0), (50, 1.0), (50, 0.95), (500, 0.999999)]      # (top-k, top-p) on 500 tokens


@pytest.mark.parametrize("top_k,top_p", POLICIES)
@pytest.mark.parametrize("draw", DRAWS)
def test_only_allowed_tokens_are_drawn(draw, top_k, top_p):
    logits, allowed = masked_rows(60, 500, 11)
    p = SamplingParams(0.7, top_k, top_p)
    got = [sample_reference(row, p, draw=draw) for row in logits]
    assert all(allowed[r, t] for r, t in enumerate(got))
    if draw == 0.0 and top_k >= 500 and top_p >= 1.0:       # in the order of ids: the first that has a probability
        assert got == [int(a.nonzero()[0]) for a in allowed]


def test_a_mask_as_a_rule_at_both_ends():
    g = torch.Generator().manual_seed(2)
    for draw in DRAWS:
        for top_k in (40, 10):
            p = SamplingParams(1.0, top_k, 1.0, allowed_tokens=[3, 5, 17])
            assert all(sample_reference(torch.randn(40, generator=g), p, draw=draw) in (3, 5, 17) for _ in range(50))
