"""Penalties, biases and masks on logits where what a call names does not fit."""

import pytest
import torch

from plain_requests import plain_rules
from test_logit_rules_gpu import make, make_mask, same

pytestmark = pytest.mark.gpu

FAR = (1 << 31) - 1


@pytest.mark.parametrize("repetition", [1.0, 1.5])
@pytest.mark.parametrize("with_tokens", [False, True])
@pytest.mark.parametrize("start,counts_as", [(13, 12), (FAR, 12), (FAR - 3, 12), (1 << 30, 12), (-1, 0), (-FAR - 1, 0)])
def test_a_start_outside_the_log_counts_as_the_nearest_place_and_is_reported(start, counts_as, with_tokens, repetition):
    from ninfer_amd_mi50_b200 import kernels
    for rows, V, capacity in ((2, 300, 16), (2, 40000, 65536), (300, 9000, 16)):      # clusters and words of two counts too
        args = make(rows, V, capacity, 16, few=9)
        args[3][1], args[5][1] = 12, torch.tensor([repetition, 0.5, 0.25])
        args[4][1] = counts_as
        tokens = torch.full((rows,), 4, dtype=torch.int32).cuda() if with_tokens else None
        args[3].clamp_(min=1)
        args[4].clamp_(max=args[3])
        want, off, h = plain_rules(*args, tokens=tokens)
        args[4][1] = start
        same(kernels.adjust_logits(*args, tokens=tokens), want, off)
        assert torch.equal(args[1].cpu(), h)
        with pytest.raises(kernels.KernelError, match="log of tokens or a mask"):
            kernels.check_status("test")
        kernels.check_status("test")


@pytest.mark.parametrize("begin,end,entries", [(FAR, FAR, 0), (FAR - 300, FAR, 0), (-5, 2, 2), (-FAR - 1, -7, 0), (2, FAR, 1), (3, 1, 0)])
def test_bias_offsets_outside_their_entries_are_reported(begin, end, entries):
    from ninfer_amd_mi50_b200 import kernels
    args = make(1, 300, 16, 16)
    ids, values = torch.tensor([5, 7, 9]).int().cuda(), torch.tensor([1.0, 2.0, 4.0]).cuda()
    first = min(max(begin, 0), 3)
    offsets = lambda lo, hi: torch.tensor([lo, hi]).int().cuda()
    want, off, _ = plain_rules(*args, bias=(offsets(first, first + entries), ids, values))
    same(kernels.adjust_logits(*args, bias=(offsets(begin, end), ids, values)), want, off)
    with pytest.raises(kernels.KernelError, match="log of tokens or a mask"):
        kernels.check_status("test")


def test_starts_and_offsets_at_the_ends_are_not_reported():
    from ninfer_amd_mi50_b200 import kernels
    args = make(3, 300, 16, 16)
    args[3][:] = torch.tensor([0, 16, 9]).int().cuda()
    args[4][:] = args[3]
    ids, values = torch.tensor([5, 7, 9]).int().cuda(), torch.tensor([1.0, 2.0, 4.0]).cuda()
    bias, mask = (torch.tensor([0, 0, 3, 3]).int().cuda(), ids, values), make_mask(300, 2, [0, -1, 1])
    want, off, _ = plain_rules(*args, bias=bias, mask=mask)
    same(kernels.adjust_logits(*args, bias=bias, mask=mask), want, off)
    kernels.check_status("test")


def test_an_out_that_overlaps_the_logits_is_refused():
    from ninfer_amd_mi50_b200 import kernels
    args = make(3, 40, 16, 16)
    buf = torch.zeros(400).cuda()
    rows = lambda at, apart: buf.as_strided((3, 40), (apart, 1), at)
    rest = args[1:]
    for logits, out in ((rows(0, 40), rows(1, 40)), (rows(0, 40), rows(0, 50)), (rows(0, 50), rows(60, 50)), (rows(40, 100), rows(0, 60))):
        with pytest.raises(ValueError, match="shares memory"):
            kernels.adjust_logits(logits, *rest, out=out)
    for logits, out in ((rows(0, 100), rows(50, 100)), (rows(0, 40), rows(120, 50)), (rows(7, 50), rows(7, 50)), (rows(140, 100), rows(100, 100))):
        logits.copy_(args[0])
        want, off, _ = plain_rules(*args)
        assert kernels.adjust_logits(logits, *rest, out=out) is out
        same(out, want, off)
    kernels.check_status("test")


def test_an_out_that_overlaps_the_rows_of_a_projection_is_refused():
    from ninfer_amd_mi50_b200 import kernels
    for dtype in (torch.float32, torch.bfloat16):
        zeros = lambda *shape: torch.zeros(shape, dtype=dtype).cuda()
        buf = zeros(64 * 64 + 64)
        x, w, a, b = buf[:64 * 64].view(64, 64), zeros(64, 64), zeros(1, 16, 64), zeros(1, 64, 16)
        scale, ids = torch.ones(1).cuda(), torch.zeros(64, dtype=torch.int32).cuda()
        for out in (x, buf[64:].view(64, 64)):
            with pytest.raises(ValueError, match="shares memory"):
                kernels.adapter_linear(x, w, a, b, scale, ids, out=out)
