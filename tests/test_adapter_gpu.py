"""Low-rank adapters beside a shared projection against the plain form in 64 bits."""

import math

import pytest
import torch

from plain_requests import outside_rounded, plain_adapter

pytestmark = pytest.mark.gpu


def make(T, K, widths, n, R, dtype, seed=0, pattern="runs"):
    g = torch.Generator().manual_seed(seed)
    N, S = sum(widths), len(widths)
    x = torch.randn(T, K, generator=g)
    w = torch.randn(N, K, generator=g) / math.sqrt(K)
    a = torch.randn(n, S * R, K, generator=g) / math.sqrt(K)
    b = torch.randn(n, N, R, generator=g) * 0.2
    scale = torch.rand(n, generator=g) + 0.5
    if pattern == "runs":            # requests of several rows, some without an adapter
        ids, t = torch.empty(T, dtype=torch.int32), 0
        while t < T:
            m = int(torch.randint(1, max(2, T // 3 + 1), (1,), generator=g))
            ids[t:t + m] = int(torch.randint(-1, n, (1,), generator=g))
            t += m
    elif pattern == "turns":         # neighbours never share one
        ids = torch.arange(T, dtype=torch.int32) % n
    elif pattern == "none":
        ids = torch.full((T,), -1, dtype=torch.int32)
    else:                            # one for all
        ids = torch.full((T,), n - 1, dtype=torch.int32)
    cast = lambda v: v.to(dtype).cuda()
    return cast(x), cast(w), cast(a), cast(b), scale.cuda(), ids.cuda()


def check(args, widths, got):
    y, off = plain_adapter(*args, widths)
    wrong = outside_rounded(got, y, off)
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()} off, first at {wrong.nonzero()[0].tolist()}"


SIZES = [
    # rows, k, widths, adapters, rank
    (1, 64, [64], 1, 16), (1, 2048, [2048], 3, 16), (2, 8, [1], 2, 16), (3, 72, [129], 4, 32), (8, 256, [64, 64, 64], 5, 16),
    (15, 200, [100, 28, 3], 4, 64), (16, 512, [384], 16, 128), (17, 512, [384], 7, 16), (33, 264, [255, 1], 40, 32),
    (64, 1024, [300, 44], 9, 16), (65, 136, [256, 256], 3, 64), (127, 192, [80], 128, 16), (128, 320, [130], 2, 128),
    (129, 320, [272, 16], 5, 16), (200, 640, [520], 6, 32), (257, 1032, [144, 300], 3, 64), (300, 128, [40, 40, 600], 11, 16),
    (513, 456, [1030], 4, 16),
    # the adapters' part as steps of a product that splits k: all members, an uneven share of rows, adapters and ranks
    (24, 520, [700], 5, 128), (41, 1000, [130, 6], 12, 64), (64, 512, [300, 140], 64, 128), (66, 1032, [1000, 72], 66, 16),
    (97, 2048, [640], 7, 32), (128, 96, [200], 3, 32), (128, 1024, [24, 8, 256], 128, 128),
    # many rows, adapters and ranks: passes of 512 rows, the last of 88 and of 28
    (600, 64, [16] * 8, 128, 128), (540, 64, [16] * 8, 128, 128),
]


@pytest.mark.parametrize("pattern", ["runs", "turns", "none", "one"])
@pytest.mark.parametrize("T,K,widths,n,R", SIZES)
def test_against_the_plain_form(T, K, widths, n, R, pattern):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, K, widths, n, R, torch.bfloat16, seed=T + K, pattern=pattern)
    check(args, widths, kernels.adapter_linear(*args, widths))
    kernels.check_status("adapter")


@pytest.mark.parametrize("T,K,widths,n,R", [(1, 64, [64], 1, 16), (5, 200, [100, 28, 3], 4, 64), (40, 513, [130], 7, 16), (130, 96, [65], 3, 32),
                                             (4, 2048, [33], 3, 16), (8, 1028, [40, 7], 4, 128), (9, 4, [1], 2, 16), (17, 3000, [66], 5, 32),
                                             (64, 8192, [30, 31], 40, 16), (65, 1024, [64], 6, 16)])
def test_float32(T, K, widths, n, R):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, K, widths, n, R, torch.float32, seed=T)
    check(args, widths, kernels.adapter_linear(*args, widths))


@pytest.mark.parametrize("T", [1, 9, 40, 150])
@pytest.mark.parametrize("K", [1, 7, 130])
def test_rows_that_are_not_16_byte_pieces(T, K):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, K, [33, 20], 3, 16, torch.bfloat16, seed=K)
    check(args, [33, 20], kernels.adapter_linear(*args, [33, 20]))


@pytest.mark.parametrize("T", [1, 16, 70, 300])
def test_more_than_one_piece_of_a_long_k(T):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, 8200, [72], 3, 16, torch.bfloat16, seed=T, pattern="turns")
    check(args, [72], kernels.adapter_linear(*args, [72]))


@pytest.mark.parametrize("T", [4, 40, 200])
def test_without_adapters_it_is_the_projection(T):
    """Rows without an adapter have the same bits whatever the pool holds and whatever their neighbours take."""
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, 512, [320], 3, 16, torch.bfloat16, pattern="none")
    alone = kernels.adapter_linear(*args)
    mixed_ids = args[5].clone()
    mixed_ids[::2] = 1
    mixed = kernels.adapter_linear(*args[:5], mixed_ids)
    assert torch.equal(alone[1::2], mixed[1::2])
    assert not torch.equal(alone[::2], mixed[::2])


@pytest.mark.parametrize("T", [3, 40, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_stays_behind_its_row(T, bad):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, 512, [320], 3, 16, torch.bfloat16, pattern="turns")
    good = kernels.adapter_linear(*args)
    x = args[0].clone()
    x[T // 2, 77] = bad
    got = kernels.adapter_linear(x, *args[1:])
    rows = torch.arange(T, device="cuda") != T // 2
    assert torch.equal(got[rows], good[rows])
    assert not torch.isfinite(got[T // 2]).any()


@pytest.mark.parametrize("T", [3, 40, 200])
@pytest.mark.parametrize("wrong", [3, 1 << 30, -5])
def test_an_adapter_outside_the_pool_is_served_as_none(T, wrong):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, 128, [96], 3, 16, torch.bfloat16, pattern="one")
    ids = args[5].clone()
    ids[T - 1] = wrong
    got = kernels.adapter_linear(*args[:5], ids)
    check((*args[:5], ids), [96], got)
    if wrong >= 0:
        with pytest.raises(kernels.KernelError, match="adapter"):
            kernels.check_status("test")
    kernels.check_status("test")


@pytest.mark.parametrize("T", [2, 40, 200])
def test_on_another_stream_and_into_a_given_tensor(T):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, 256, [128], 2, 16, torch.bfloat16)
    want = kernels.adapter_linear(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = args[0] * 2                     # made on that stream right before
        x = x / 2
        out = torch.full((T, 128), math.nan, dtype=torch.bfloat16, device="cuda")
        assert kernels.adapter_linear(x, *args[1:], out=out) is out
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


@pytest.mark.parametrize("T", [1, 8, 40, 200])
def test_the_same_bits_every_time_and_out_of_a_graph(T):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, 1024, [256, 64], 4, 32, torch.bfloat16, pattern="turns")
    want = kernels.adapter_linear(*args, [256, 64])
    for _ in range(5):
        assert torch.equal(kernels.adapter_linear(*args, [256, 64]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.adapter_linear(*args, [256, 64])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.adapter_linear(*args, [256, 64])
    graph.replay()
    assert torch.equal(got, want)
    args[5].fill_(-1)                       # the graph serves whichever adapters its tensor names
    graph.replay()
    assert torch.equal(got, kernels.adapter_linear(*args, [256, 64]))


def test_no_rows():
    from ninfer_amd_mi50_b200 import kernels
    args = make(4, 64, [48], 2, 16, torch.bfloat16)
    assert kernels.adapter_linear(args[0][:0], *args[1:5], args[5][:0]).shape == (0, 48)


def test_refusals():
    from ninfer_amd_mi50_b200 import kernels
    x, w, a, b, s, ids = make(4, 64, [48], 2, 16, torch.bfloat16)
    f = kernels.adapter_linear
    bad = [
        (x[:, :56].contiguous(), w, a, b, s, ids), (x, w[:, :56].contiguous(), a, b, s, ids), (x, w, a[:, :8].contiguous(), b, s, ids),
        (x, w, a, b[:, :40].contiguous(), s, ids), (x, w, a, b[:, :, :8].contiguous(), s, ids), (x, w, a, b, s[:1], ids),
        (x, w, a, b, s, ids[:3]), (x.t(), w, a, b, s, ids), (x[:, ::2], w, a, b, s, ids), (x[0], w, a, b, s, ids),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            f(*args)
    for args in [(x, w.float(), a, b, s, ids), (x, w, a.float(), b, s, ids), (x, w, a, b, s.bfloat16(), ids), (x, w, a, b, s, ids.long()),
                 (x.half(), w.half(), a.half(), b.half(), s, ids)]:
        with pytest.raises(TypeError):
            f(*args)
    for widths in ([40], [40, 9], [48, 0], [], [6] * 8 + [0]):
        with pytest.raises(ValueError):
            f(x, w, a, b, s, ids, widths)
    with pytest.raises(ValueError):
        f(x, w, a, b, s, ids, out=torch.empty(4, 47, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        f(x, w, a, b, s, ids.cpu())
    with pytest.raises(kernels.KernelError):
        f(*(t.cpu() for t in (x, w, a, b, s, ids)))
