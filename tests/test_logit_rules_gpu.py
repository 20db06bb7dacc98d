"""Penalties, biases and masks on logits, over logs of tokens on the device, against the plain form in 64 bits."""

import math
import random

import pytest
import torch

from plain_requests import plain_rules

pytestmark = pytest.mark.gpu


def make(R, V, capacity, longest, seed=0, few=None):
    """Logits, a log and its rows; tokens among the first `few` of the vocabulary, so that they occur again and again."""
    g, rnd = torch.Generator().manual_seed(seed), random.Random(seed)
    logits = torch.randn(R, V, generator=g) * 3
    history = torch.randint(0, min(V, few or V), (R + 3, capacity), generator=g).int()
    lengths = torch.tensor([longest] + [rnd.randint(1, longest) for _ in range(R - 1)], dtype=torch.int32)
    starts = torch.tensor([rnd.randint(0, int(n)) for n in lengths], dtype=torch.int32)
    slots = torch.tensor(rnd.sample(range(R + 3), R), dtype=torch.int32)
    pen = torch.tensor([[rnd.choice([1.0, 1.05, 1.3, 0.8]), rnd.choice([0.0, 0.3]), rnd.choice([0.0, 0.7, -0.2])] for _ in range(R)])
    return [t.cuda() for t in (logits, history, slots, lengths, starts, pen)]


def make_bias(R, V, most, seed=0):
    rnd = random.Random(seed)
    per = [rnd.sample(range(V), rnd.randint(0, min(V, most))) for _ in range(R)]
    offsets = [0]
    for p in per:
        offsets.append(offsets[-1] + len(p))
    ids = torch.tensor([i for p in per for i in p], dtype=torch.int32)
    values = torch.tensor([rnd.choice([-100.0, 2.5, 0.1, -math.inf]) for _ in ids])
    return torch.tensor(offsets, dtype=torch.int32).cuda(), ids.cuda(), values.cuda()


def make_mask(V, M, index, keep=0.5, seed=0):
    g = torch.Generator().manual_seed(seed)
    words = (V + 31) // 32
    allowed = torch.rand(M, words, 32, generator=g) < keep
    bits = (allowed.long() << torch.arange(32)).sum(-1)
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
    return bits.cuda(), torch.tensor(index, dtype=torch.int32).cuda()


def same(got, want, off):
    got = got.cpu().double()
    special = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    both = special & ~torch.isnan(want)
    assert torch.equal(got[both], want[both])
    fine = ~special
    wrong = fine & ~((got - want).abs() <= off)
    assert not wrong.any(), f"{int(wrong.sum())} off, first {wrong.nonzero()[0].tolist()}: {got[wrong][0]} for {want[wrong][0]}"


@pytest.mark.parametrize("R,V,capacity,longest,few", [
    (1, 1, 4, 1, None), (1, 3, 4, 4, None), (2, 31, 16, 9, None), (3, 33, 8, 8, 5), (5, 1000, 64, 50, 20), (2, 2048, 64, 64, None),
    (4, 2049, 512, 512, 30), (3, 4099, 2048, 2047, 300), (1, 32003, 1024, 1000, None), (2, 151936, 128, 100, None),
    (40, 131075, 64, 60, 30), (75, 16385, 128, 128, 50), (20, 131071, 65536, 300, 40), (3, 5000, 65536, 66000 - 465, 700),
    (2, 40001, 70000, 70000, None), (3, 8189, 65536, 16384, 8000), (1, 8195, 65540, 16385, None), (4, 151936, 65536, 40000, 30000)])
@pytest.mark.parametrize("what", ["penalties", "bias", "mask", "all"])
def test_against_the_plain_form(R, V, capacity, longest, few, what):
    from ninfer_amd_mi50_b200 import kernels
    args = make(R, V, capacity, longest, seed=V, few=few)
    bias = make_bias(R, V, 40, V) if what in ("bias", "all") else None
    mask = make_mask(V, 2, [r % 3 - 1 for r in range(R)], seed=V) if what in ("mask", "all") else None
    if what in ("bias", "mask"):
        args[5] = torch.tensor([[1.0, 0.0, 0.0]] * R).cuda()
    want, off, _ = plain_rules(*args, bias=bias, mask=mask)
    before = args[0].clone()
    got = kernels.adjust_logits(*args, bias=bias, mask=mask)
    same(got, want, off)
    assert torch.equal(args[0], before)
    into = args[0].clone()
    assert kernels.adjust_logits(into, *args[1:], bias=bias, mask=mask, out=into) is into
    assert torch.equal(into, got)
    kernels.check_status("rules")


@pytest.mark.parametrize("R,V", [(1, 100), (4, 1001), (9, 5000)])
def test_the_last_tokens_go_into_the_log(R, V):
    from ninfer_amd_mi50_b200 import kernels
    args = make(R, V, 64, 60, seed=R, few=12)
    args[3][-1] = 1                                             # a log of nothing but its new token
    args[4][-1] = 0
    tokens = torch.randint(0, 12, (R,), dtype=torch.int32).cuda()
    want, off, log = plain_rules(*args, tokens=tokens)
    got = kernels.adjust_logits(*args, tokens=tokens)
    same(got, want, off)
    assert torch.equal(args[1].cpu(), log)
    assert torch.equal(kernels.adjust_logits(*args), got)       # the log holds them now


@pytest.mark.parametrize("length", [16384, 16385, 30001])
def test_the_last_token_of_a_long_log(length):
    from ninfer_amd_mi50_b200 import kernels
    args = make(2, 20003, 65536, length, seed=length, few=15000)
    args[3][1] = length - 7
    tokens = torch.tensor([14999, 8191], dtype=torch.int32).cuda()
    full = args[1].clone()
    full[args[2].long(), args[3].long() - 1] = tokens
    want, off, _ = plain_rules(args[0], full, *args[2:])
    got = kernels.adjust_logits(*args, tokens=tokens)
    same(got, want, off)
    assert torch.equal(args[1], full)


def test_append_history():
    from ninfer_amd_mi50_b200 import kernels
    log = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    kernels.append_history(log, ints(0, 0, 2, -1, 1), ints(0, 1, 7, 3, 4), ints(5, 6, 7, 8, 9))
    want = torch.full((3, 8), -1, dtype=torch.int32)
    want[0, 0], want[0, 1], want[2, 7], want[1, 4] = 5, 6, 7, 9
    assert torch.equal(log.cpu(), want)
    kernels.check_status("append")
    kernels.append_history(log, ints(3, 1), ints(0, 8), ints(1, 1))
    assert torch.equal(log.cpu(), want)
    with pytest.raises(kernels.KernelError, match="log of tokens"):
        kernels.check_status("append")
    kernels.append_history(log, log[0, :0], log[0, :0], log[0, :0])


def test_no_tokens_yet():
    from ninfer_amd_mi50_b200 import kernels
    args = make(2, 500, 8, 8)
    args[3].zero_(); args[4].zero_()
    assert torch.equal(kernels.adjust_logits(*args), args[0])
    kernels.check_status("rules")


@pytest.mark.parametrize("V", [37, 3000])
def test_values_that_are_not_finite(V):
    from ninfer_amd_mi50_b200 import kernels
    args = make(3, V, 64, 64, few=V)
    odd = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 3e38, -3e38, 1e-44])
    args[0][:, :8] = odd.cuda()
    args[1][:, :32] = torch.arange(8).repeat(4).int().cuda()    # each of them four times
    args[3].fill_(64)
    args[5] = torch.tensor([[1.3, 0.5, 0.1], [0.5, 0.0, 0.0], [40.0, 0.0, 0.0]]).cuda()
    mask = make_mask(V, 1, [0, -1, 0])
    mask[0][0, 0] = 0b1010_1010 - 256                           # tokens 0, 2, 4, 6 not allowed
    want, off, _ = plain_rules(*args, mask=mask)
    same(kernels.adjust_logits(*args, mask=mask), want, off + 1e-38)


def test_many_occurrences_overflow_as_repeated_products_do():
    from ninfer_amd_mi50_b200 import kernels
    logits = torch.tensor([[2.0, -2.0, 0.0, 5.0]]).cuda()
    log = torch.tensor([[0, 1, 2] * 1000]).int().cuda()
    one = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")
    got = kernels.adjust_logits(logits, log, one(0), one(3000), one(0), torch.tensor([[1.5, 0.0, 0.0]]).cuda())
    assert got.cpu().tolist() == [[0.0, -math.inf, 0.0, 5.0]]


def test_a_mask_that_allows_nothing():
    from ninfer_amd_mi50_b200 import kernels
    args = make(2, 777, 16, 16)
    args[0][0, 5] = math.nan
    bits = torch.zeros((1, 25), dtype=torch.int32, device="cuda")
    got = kernels.adjust_logits(*args, mask=(bits, torch.tensor([0, -1], dtype=torch.int32).cuda()))
    assert (got[0] == -math.inf).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("ld", [1000, 1001, 1003, 1024])
@pytest.mark.parametrize("first", [0, 1])
def test_rows_further_apart_and_off_their_boundaries(ld, first):
    from ninfer_amd_mi50_b200 import kernels
    args = make(4, 999, 64, 60, few=50)
    wide = torch.zeros(4, ld + 4, device="cuda")[:, first:first + 999]
    wide.copy_(args[0])
    mask, bias = make_mask(999, 2, [0, 1, -1, 0]), make_bias(4, 999, 20)
    want = kernels.adjust_logits(*args, mask=mask, bias=bias)
    assert torch.equal(kernels.adjust_logits(wide, *args[1:], mask=mask, bias=bias), want)
    out = torch.full((4, ld + 2), 7.0, device="cuda")
    kernels.adjust_logits(wide, *args[1:], mask=mask, bias=bias, out=out[:, 1:1000])
    assert torch.equal(out[:, 1:1000], want) and (out[:, 0] == 7).all() and (out[:, 1000:] == 7).all()
    kernels.adjust_logits(wide, *args[1:], mask=mask, bias=bias, out=wide)
    assert torch.equal(wide, want)


def test_tokens_outside_the_vocabulary_count_nowhere():
    from ninfer_amd_mi50_b200 import kernels
    args = make(2, 50, 16, 16)
    args[1][:, ::2] = torch.tensor([50, -1, 1 << 30, -(1 << 31)] * 2).int().cuda()
    want, off, _ = plain_rules(*args)
    same(kernels.adjust_logits(*args), want, off)


@pytest.mark.parametrize("field,value", [("slot", 99), ("slot", -1), ("length", 17), ("length", -1), ("mask", 2)])
def test_what_does_not_fit_is_reported_and_changes_its_row_as_if_it_were_not_there(field, value):
    from ninfer_amd_mi50_b200 import kernels
    args = make(2, 300, 16, 16, few=9)
    mask = make_mask(300, 2, [0, 1])
    good = kernels.adjust_logits(*args, mask=mask)
    if field == "mask":
        mask[1][1] = value
        want = kernels.adjust_logits(*(t[1:] if i != 1 else t for i, t in enumerate(args)))
    else:
        args[2 if field == "slot" else 3][1] = value
        want = args[0][1:].clone()
        allowed = ((mask[0][1][:, None] >> torch.arange(32, device="cuda").int()) & 1).flatten()[:300] > 0
        want[0, ~allowed] = -math.inf
    got = kernels.adjust_logits(*args, mask=mask)
    assert torch.equal(got[0], good[0]) and torch.equal(got[1:], want)
    with pytest.raises(kernels.KernelError, match="log of tokens or a mask"):
        kernels.check_status("test")


def test_on_another_stream():
    from ninfer_amd_mi50_b200 import kernels
    args = make(6, 20000, 64, 60)
    want = kernels.adjust_logits(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logits = args[0] + 1
        logits -= 1
        got = kernels.adjust_logits(args[0].clone(), *args[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_nothing_to_do():
    from ninfer_amd_mi50_b200 import kernels
    args = make(2, 40, 8, 8)
    none = [t[:0] if i != 1 else t for i, t in enumerate(args)]
    assert kernels.adjust_logits(*none).shape == (0, 40)


def test_refusals():
    from ninfer_amd_mi50_b200 import kernels
    l, h, s, n, st, p = make(3, 100, 16, 16)
    f = kernels.adjust_logits
    for args in [(l[0], h, s, n, st, p), (l, h[0], s, n, st, p), (l, h, s[:2], n, st, p), (l, h, s, n[:2], st, p), (l, h, s, n, st[:2], p),
                 (l, h, s, n, st, p[:, :2].contiguous()), (l[:, ::2], h, s, n, st, p), (l, h[:, :15].contiguous(), s, n, st, p),
                 (l, h[:, ::2], s, n, st, p), (l[:1].expand(3, 100), h, s, n, st, p)]:
        with pytest.raises(ValueError):
            f(*args)
    for args in [(l.bfloat16(), h, s, n, st, p), (l, h.long(), s, n, st, p), (l, h, s.long(), n, st, p), (l, h, s, n, st, p.double())]:
        with pytest.raises(TypeError):
            f(*args)
    bias, (bits, index) = make_bias(3, 100, 5), make_mask(100, 1, [0, 0, 0])
    for more in [dict(bias=(bias[0][:3], bias[1], bias[2])), dict(bias=(bias[0], bias[1], bias[2][:-1])), dict(mask=(bits[:, :3], index)),
                 dict(mask=(bits, index[:2])), dict(mask=(bits[0], index)), dict(tokens=s[:2]), dict(out=l[:2]), dict(tokens=s.cpu())]:
        with pytest.raises((ValueError, kernels.KernelError)):
            f(l, h, s, n, st, p, **more)
    with pytest.raises(TypeError):
        f(l, h, s, n, st, p, mask=(bits.long(), index))
    with pytest.raises(kernels.KernelError):
        f(*(t.cpu() for t in (l, h, s, n, st, p)))
    with pytest.raises(ValueError):
        kernels.append_history(h, s, n, st[:2])
    with pytest.raises(TypeError):
        kernels.append_history(h, s.long(), n, st)
