"""Draws from rows with masks on the device: never a token of probability 0, and what the host twin draws away from roundings."""

import pytest
import torch

from draw_cases import DRAWS, masked_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [2, 3, 500, 1024, 5003, 40000])
@pytest.mark.parametrize("whole", [True, False])
def test_only_allowed_tokens_are_drawn(V, whole):
    from ninfer_amd_mi50_b200 import kernels
    from ninfer_amd_mi50_b200.sampling import SamplingParams, sample_reference
    rows = 48
    logits, allowed = (masked_rows(rows, V, V) if V > 3 else
                       (torch.tensor([[0.0, -float("inf")], [-float("inf"), 1.0]]).repeat(rows // 2, 1) if V == 2 else
                        torch.tensor([[-float("inf"), 2.0, -float("inf")]]).repeat(rows, 1), None))
    allowed = logits > -float("inf") if allowed is None else allowed
    for top_k, top_p in [(V, 1.0)] if whole else [(min(V, 50), 1.0), (min(V, 50), 0.95), (min(V, 1024), 0.999999)]:
        for draw in DRAWS + (0.37,):
            full = lambda v, dt: torch.full((rows,), v, dtype=dt).cuda()
            got = kernels.sample_rows(logits.cuda(), full(0.7, torch.float32), full(top_k, torch.int32), full(top_p, torch.float32),
                                      full(draw, torch.float32)).cpu()
            assert allowed[torch.arange(rows), got.long()].all(), (top_k, top_p, draw)
            if draw == 0.0:                             # no rounding has a say in the first one
                p = SamplingParams(0.7, top_k, top_p)
                assert got.tolist() == [sample_reference(row, p, draw=draw) for row in logits]
