"""Trees of drafted tokens where a call goes from one piece of work to the next, or its operands do not fit, against plain
forms in 64 bits."""

import pytest
import torch

from ninfer_amd_mi50_b200 import kernels
from ninfer_amd_mi50_b200.kernels import drafts
from plain_drafts import make_attention, plain_attention
from test_drafts_gpu import attend, near

pytestmark = pytest.mark.gpu


@pytest.fixture
def asked():
    """asked(form): the form of attention that calls have from here on."""
    def ask(form):
        kernels.TUNING["tree_attention"] = form
    yield ask
    kernels.TUNING["tree_attention"] = "auto"


def form_of(c, heads, page_size):
    """The form that serves the last call of these sizes, by its plan."""
    plan = [p for key, (p, _) in drafts._plans.items() if key[:6] == (len(c["lengths"]), c["qkv"].shape[0], *heads, page_size)
            and key[8] == c["longest"] and key[-1] == kernels.TUNING["tree_attention"]]
    return plan[-1] & 3


@pytest.mark.parametrize("heads", [(8, 8, 128), (6, 6, 64)])
def test_one_tile_of_rows_after_the_other_with_keys_that_rise_at_once(heads, asked):
    """Each CTA has several items of one tile of rows, whose sums both groups of rows read, and every block's second 64 keys
    stand far above its first 64, the first block's of an item too: 16 in the natural exponent, 23 in that of the weights."""
    asked(1)
    sizes, lengths = [5 + 7 * s % 20 for s in range(48)], [130 + 29 * s % 270 for s in range(48)]
    c = make_attention(sizes, lengths, heads, 64, seed=5)
    q, pages = c["qkv"].clone(), c["pages"].clone()
    q[:, :heads[0] * heads[2]:heads[2]] = 4.0                # the first dimension carries a score of its own
    for s, n in enumerate(sizes):
        for p in range(-(-(lengths[s] + n) // 64)):
            pages[c["table"][s, p].long(), 0, :, :, 0] = (16.0 if p % 2 else 0.0) / 4 / 0.1
    c["qkv"], c["pages"] = q.bfloat16().float(), pages.bfloat16().float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], 64, c["lengths"], c["row0"], c["mask"], 0.1)
    first = attend(c, heads, 64, torch.bfloat16, 0.1)
    assert form_of(c, heads, 64) == 1
    # (weights of the first 64 may be rounded twice: see test_scores_that_rise_within_a_block_of_keys)
    near(first, want, weight * 1.25, size, c["longest"], torch.bfloat16, heads[2])
    for _ in range(20):
        assert torch.equal(attend(c, heads, 64, torch.bfloat16, 0.1), first)
    kernels.check_status()
