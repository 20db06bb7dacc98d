"""Trees of drafted tokens: attention over the cache, verification, rows moved and pages copied, against plain forms in 64 bits."""

import math
import random

import pytest
import torch

from ninfer_amd_mi50_b200 import kernels
from plain_drafts import block_tables, make_attention, make_verify, plain_attention, plain_compact, plain_verify

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def attend(c, heads, page_size, dtype, scale, out=None, qkv=None):
    qkv = c["qkv"].to(dtype).cuda() if qkv is None else qkv
    return kernels.tree_attention(qkv, *heads, c["pages"].to(dtype).cuda(), c["table"].cuda(), page_size, ints(c["lengths"]), ints(c["row0"]),
                                  c["mask"].cuda(), c["longest"], scale, out=out)


@pytest.fixture(params=["auto", 1, 2], ids=["auto", "tcgen05", "mma"])
def form(request):
    """The forms of the bfloat16 attention, each for every size that it takes."""
    kernels.TUNING["tree_attention"] = request.param
    yield request.param
    kernels.TUNING["tree_attention"] = "auto"


def taken(form, heads, page_size, dtype=torch.bfloat16):
    return form == "auto" or (dtype == torch.bfloat16 and heads[2] in (64, 128) and page_size % 16 == 0 and (form == 2 or page_size in (16, 32, 64, 128)))


def near(got, want, weight, size, keys, dtype, D):
    """The result's rounding is half a step of its size.  A weight is off by what its score and the largest one are off by,
    each (D + 2) roundings of half a step of float32 of the sum of |q||k|, by two steps of the exponential, and in bfloat16
    by its own rounding, half a step; sums over keys by a rounding of float32 for each of them and for a merge of shares."""
    half = torch.finfo(dtype).eps / 2
    f = 2.0 ** -24
    off = 2 * (D + 2) * f * size + 8 * f + 2 * (keys + 64) * f + (half if dtype == torch.bfloat16 else 0.0)
    bound = half * want.abs() + off * weight * (1 + half) + 1e-30
    wrong = ~((got.double().cpu() - want).abs() <= bound)
    assert not wrong.any(), f"{int(wrong.sum())} off, first {wrong.nonzero()[0].tolist()}: {got.cpu()[wrong][0]} for {want[wrong][0]} +- {bound[wrong][0]}"


SIZES = [
    # nodes of each request, keys that each held, heads, page size
    ([1], [0], (1, 1, 16), 16),
    ([1], [1], (2, 1, 64), 16),
    ([5], [0], (4, 2, 64), 16),
    ([8], [300], (4, 4, 128), 64),
    ([7, 1, 13], [15, 16, 17], (4, 2, 128), 16),
    ([3, 0, 4], [40, 9, 0], (6, 2, 48), 32),
    ([31, 32, 33], [127, 128, 129], (4, 2, 64), 64),
    ([64], [95], (7, 1, 128), 64),
    ([20, 3], [500, 1200], (28, 4, 128), 64),
    ([100], [33], (2, 2, 32), 64),
    ([129, 2], [200, 700], (2, 1, 128), 128),
    ([256], [64], (3, 1, 64), 32),
    ([9, 4], [70, 1], (4, 1, 256), 16),
    ([6], [50], (3, 3, 80), 7),
    ([11], [1030], (2, 2, 128), 96),
    ([17], [63], (24, 1, 64), 64),
    ([2], [2500], (16, 16, 64), 64),
    ([40], [4000], (2, 1, 64), 32),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_attention(case, dtype, form):
    sizes, lengths, heads, ps = SIZES[case]
    if not taken(form, heads, ps, dtype):
        return
    c = make_attention(sizes, lengths, heads, ps, seed=case, shape="chain" if case % 3 == 0 else "tree", sharp=1.0 + case % 2)
    c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
    scale = 1 / math.sqrt(heads[2])
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], ps, c["lengths"], c["row0"], c["mask"], scale)
    near(attend(c, heads, ps, dtype, scale), want, weight, size, c["longest"], dtype, heads[2])
    kernels.check_status()


@pytest.mark.parametrize("heads,most,page_size", [((8, 8, 128), 40, 64), ((8, 8, 64), 40, 16), ((24, 2, 128), 40, 64), ((24, 2, 64), 30, 32), ((5, 1, 128), 64, 128)])
def test_many_requests_of_many_lengths(heads, most, page_size, form):
    """More work than there are SMs: each goes from request to request, with one tile of rows and with two."""
    for seed in range(3):
        rnd = random.Random(seed)
        sizes = [rnd.randint(0 if s else 1, most) for s in range(30)]
        lengths = [rnd.choice([0, 1, 127, 128, rnd.randint(0, 900), rnd.randint(0, 300)]) for _ in sizes]
        lengths[5] = 2000
        c = make_attention(sizes, lengths, heads, page_size, seed=seed, words=2)
        c["qkv"], c["pages"] = c["qkv"].bfloat16().float(), c["pages"].bfloat16().float()
        got = attend(c, heads, page_size, torch.bfloat16, 0.1)
        kernels.check_status()
        kernels.TUNING["tree_attention"] = "auto"
        want = attend(c, heads, page_size, torch.float32, 0.1).double()
        kernels.TUNING["tree_attention"] = form
        # (against the float32 form, which the plain one was compared with: a weight's rounding and the result's, of values below 6)
        assert float((got.double() - want).abs().max()) <= 6 * 2.0 ** -8 * 2 + 1e-4
        for s in rnd.sample(range(30), 4):        # and some requests against the plain form
            lo, hi = c["row0"][s:s + 2]
            one, weight, size = plain_attention(c["qkv"][lo:hi], *heads, c["pages"], c["table"][s:s + 1], page_size, [lengths[s]], [0, hi - lo], c["mask"][lo:hi], 0.1)
            near(got[lo:hi], one, weight, size, c["longest"], torch.bfloat16, heads[2])


@pytest.mark.parametrize("spikes", [(), (64,), (0, 64), (63, 127), (31, 32, 95, 96), (10, 70, 129, 200, 300, 301)], ids=str)
@pytest.mark.parametrize("slope", [0.0, 0.25, -0.25])
def test_scores_that_rise_within_a_block_of_keys(slope, spikes, form):
    """Scores that climb from key to key, and keys that stand 16 to 48 above the ones before them."""
    heads, ps = (8, 1, 128), 64
    c = make_attention([6, 20], [320, 61], heads, ps, seed=3, shape="chain")
    q, pages = c["qkv"].clone(), c["pages"].clone()
    q[:, :heads[0] * 128:128] = 4.0                          # the first dimension carries a score of its own
    for s in range(2):
        n = c["row0"][s + 1] - c["row0"][s]
        for j in range(c["lengths"][s] + n):
            high = slope * j + sum(16.0 * (1 + i % 3) for i, k in enumerate(spikes) if k == j)
            pages[c["table"][s, j // ps].long(), 0, :, j % ps, 0] = high / 4 / 0.1
    c["qkv"], c["pages"] = q.bfloat16().float(), pages.bfloat16().float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], ps, c["lengths"], c["row0"], c["mask"], 0.1)
    # A weight that a later key of its block makes less than 2^-8 of the largest may be rounded twice: 64 of them come to at
    # most a quarter of the sum, so that much of half a step more.
    near(attend(c, heads, ps, torch.bfloat16, 0.1), want, weight * 1.25, size, c["longest"], torch.bfloat16, 128)
    kernels.check_status()


def test_more_requests_than_a_launch_takes(form):
    heads, ps, n = (4, 2, 64), 16, 1100
    rnd = random.Random(4)
    sizes = [rnd.randint(0, 3) for _ in range(n)]
    sizes[511], sizes[512], sizes[1099] = 3, 2, 1
    lengths = [rnd.randint(0, 40) for _ in range(n)]
    c = make_attention(sizes, lengths, heads, ps, seed=6)
    c["qkv"], c["pages"] = c["qkv"].bfloat16().float(), c["pages"].bfloat16().float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], ps, c["lengths"], c["row0"], c["mask"], 0.2)
    near(attend(c, heads, ps, torch.bfloat16, 0.2), want, weight, size, c["longest"], torch.bfloat16, 64)
    kernels.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_more_requests_and_heads_than_a_dimension_of_a_grid(dtype, form):
    heads, ps, n = (8, 8, 64), 16, 9000
    if not taken(form, heads, ps, dtype):
        return
    sizes, lengths = [0] * n, [0] * n
    for s in (0, 1, 511, 512, 8190, 8191, 8192, 8999):
        sizes[s], lengths[s] = 1 + s % 3, 5 + s % 40
    c = make_attention(sizes, lengths, heads, ps, seed=8)
    c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], ps, c["lengths"], c["row0"], c["mask"], 0.2)
    near(attend(c, heads, ps, dtype, 0.2), want, weight, size, c["longest"], dtype, 64)
    kernels.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,length", [((4, 2, 64), 0), ((8, 1, 128), 37), ((2, 2, 48), 130), ((16, 1, 128), 600)])
def test_any_mask_and_rows_that_see_nothing(heads, length, dtype, form):
    if not taken(form, heads, 16, dtype):
        return
    sizes = [21, 40]
    c = make_attention(sizes, [length, 0], heads, 16, seed=5)
    g = torch.Generator().manual_seed(1)
    c["mask"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (61, 2), generator=g).int()         # (bits of nodes that a request has not, too)
    c["mask"][[0, 20, 21, 50, 60]] = 0
    c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], 16, c["lengths"], c["row0"], c["mask"], 0.2)
    assert not want[[21, 50, 60]].any()
    near(attend(c, heads, 16, dtype, 0.2), want, weight, size, c["longest"], dtype, heads[2])
    kernels.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,length", [((4, 2, 64), 17), ((8, 1, 128), 700), ((2, 1, 32), 100)])
def test_rows_without_a_request_stay_and_what_lies_behind_the_nodes_is_not_looked_at(heads, length, dtype, form):
    if not taken(form, heads, 16, dtype):
        return
    c = make_attention([5, 9, 3], [length, 3, length], heads, 16, seed=2)
    c["row0"] = [0, 5, 14, 14]                                # the last rows belong to nobody
    c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], 16, c["lengths"], c["row0"], c["mask"], 0.1)
    last = {}
    for s in (0, 1):
        end = c["lengths"][s] + c["row0"][s + 1] - c["row0"][s]
        if end % 16:
            c["pages"][c["table"][s, end // 16].long(), :, :, end % 16:] = math.nan
            last[s] = end
    assert last
    out = torch.full((17, heads[0] * heads[2]), 7.0, dtype=dtype, device="cuda")
    got = attend(c, heads, 16, dtype, 0.1, out=out)
    assert got is out and bool((out[14:] == 7).all())
    near(out[:14], want[:14], weight[:14], size, c["longest"], dtype, heads[2])
    kernels.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_queries_of_rows_that_lie_apart(dtype):
    heads = (6, 2, 64)
    c = make_attention([9, 30], [50, 333], heads, 32, seed=3)
    c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], 32, c["lengths"], c["row0"], c["mask"], 0.125)
    wide = torch.full((39, 2 * c["qkv"].shape[1] + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 3:3 + c["qkv"].shape[1]] = c["qkv"].to(dtype)
    for view in (wide[:, 3:3 + heads[0] * 64], wide[:, 3:3 + c["qkv"].shape[1]]):
        near(attend(c, heads, 32, dtype, 0.125, qkv=view), want, weight, size, c["longest"], dtype, 64)


@pytest.mark.parametrize("dtype,heads,pool", [(torch.bfloat16, (4, 2, 128), 80000), (torch.float32, (4, 2, 128), 40000), (torch.bfloat16, (4, 2, 48), 200000)],
                         ids=["bf16", "f32", "bf16 of 48"])
def test_pages_more_than_four_gigabytes_apart(dtype, heads, pool, form):
    if not taken(form, heads, 64, dtype):
        return
    c = make_attention([5, 33], [300, 70], heads, 64, seed=9)
    c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], 64, c["lengths"], c["row0"], c["mask"], 0.1)
    n = c["pages"].shape[0]
    pages = torch.empty((pool, *c["pages"].shape[1:]), dtype=dtype, device="cuda")
    assert pages.nbytes > 4 << 30
    at = torch.cat([torch.arange(n - n // 2) * 2, pool - 1 - torch.arange(n // 2)])         # both ends of the pool
    pages[at.cuda()] = c["pages"].to(dtype).cuda()
    table = torch.where(c["table"] >= 0, at[c["table"].long().clamp_min(0)], -1).int().cuda()
    got = kernels.tree_attention(c["qkv"].to(dtype).cuda(), *heads, pages, table, 64, ints(c["lengths"]), ints(c["row0"]), c["mask"].cuda(), c["longest"], 0.1)
    near(got, want, weight, size, c["longest"], dtype, heads[2])
    # and rows and pages copied there
    first, last = pages[0].clone(), pages[pool - 1].clone()
    kernels.copy_pages(pages, ints([0, pool - 1]), ints([pool - 2, 2 * n]))
    assert torch.equal(pages[pool - 2], first) and torch.equal(pages[2 * n], last)
    kernels.compact_cache(pages, ints([[pool - 1]]), ints([3]), ints([[4, 9]]), ints([2]))
    last[:, :, 4], last[:, :, 5] = last[:, :, 7].clone(), last[:, :, 12].clone()
    assert torch.equal(pages[pool - 1], last)
    kernels.check_status()


def test_two_calls_at_once_on_streams_of_their_own(form):
    """Neither waits for the other, and each has the bits that it has alone."""
    cases = [make_attention([40, 64, 9], [900, 300, 2000], (8, 2, 128), 64, seed=1), make_attention([30, 2], [1500, 700], (8, 2, 128), 64, seed=2)]
    args = [((c["qkv"].bfloat16().cuda(), 8, 2, 128, c["pages"].bfloat16().cuda(), c["table"].cuda(), 64, ints(c["lengths"]), ints(c["row0"]),
              c["mask"].cuda(), c["longest"], 0.1)) for c in cases]
    v = make_verify([5, 40], 30000, True, seed=3)
    v = {k: x.cuda() if isinstance(x, torch.Tensor) else x for k, x in v.items()}
    check = lambda: kernels.verify_drafts(v["probs"], v["tokens"], v["parents"], ints(v["row0"]), v["draws"], 8, v["draft"])
    alone = [kernels.tree_attention(*x) for x in args] + list(check())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        got = []
        for s, x in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(kernels.tree_attention(*x))
        with torch.cuda.stream(streams[2]):
            got += check()
        torch.cuda.synchronize()
        for x, y in zip(got, alone):
            assert torch.equal(x, y)
    kernels.check_status()


def test_a_loose_bound_and_other_requests_change_little():
    """What max_context allows beyond the real lengths only changes how keys are shared out."""
    heads = (8, 2, 128)
    c = make_attention([12, 12], [900, 41], heads, 64, seed=9)
    near_bits = [attend({**c, "longest": m}, heads, 64, torch.float32, 0.09) for m in (c["longest"], 4096, 100000)]
    for v in near_bits[1:]:
        torch.testing.assert_close(v, near_bits[0], rtol=2e-5, atol=2e-5)
    kernels.check_status()


def test_same_bits_every_time():
    heads = (28, 4, 128)
    c = make_attention([33, 60], [3000, 1111], heads, 64, seed=4)
    for form, dtype in (("auto", torch.float32), (0, torch.bfloat16), (1, torch.bfloat16), (2, torch.bfloat16)):
        kernels.TUNING["tree_attention"] = form
        first = attend(c, heads, 64, dtype, 0.09)
        assert all(torch.equal(first, attend(c, heads, 64, dtype, 0.09)) for _ in range(5))
    kernels.TUNING["tree_attention"] = "auto"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_pages_outside_the_pool_and_rows_that_do_not_fit_are_reported(dtype, form):
    heads = (4, 2, 64)
    if not taken(form, heads, 16, dtype):
        return
    for what in ("page", "page beyond", "context", "row0", "length", "table"):
        c = make_attention([4, 6], [40, 90], heads, 16, seed=6)
        if what == "page":
            c["table"][1, 2] = -1
        if what == "page beyond":
            c["table"][0, 0] = 10 ** 6
        if what == "context":
            c["longest"] = 64
        if what == "row0":
            c["row0"] = [0, 4, 99]
        if what == "length":
            c["lengths"] = [-3, 90]
        if what == "table":
            c["table"] = c["table"][:, :3].contiguous()
        attend(c, heads, 16, dtype, 0.1)
        with pytest.raises(kernels.KernelError, match="tree of drafted"):
            kernels.check_status()
    kernels.check_status()


def test_refusals_of_attention():
    heads = (4, 2, 64)
    c = make_attention([4], [20], heads, 16)
    args = [c["qkv"].cuda(), *heads, c["pages"].cuda(), c["table"].cuda(), 16, ints(c["lengths"]), ints(c["row0"]), c["mask"].cuda(), 24, 0.1]
    kernels.tree_attention(*args)
    T = 4
    for at, bad in [(0, args[0].cpu()), (0, args[0].half()), (0, args[0].bfloat16()), (0, args[0].t()), (0, args[0][0]), (0, args[0][:, :200]), (1, 3), (1, 0),
                    (2, 0), (3, 40), (3, 272), (4, args[4][:, :1]), (4, args[4].transpose(2, 3)), (4, args[4].flatten()[1:1 + 16 * 64 * 4].view(1, 2, 2, 16, 64)),
                    (5, args[5].long()), (5, args[5][:0]), (5, args[5][0]), (5, args[5].cpu()), (6, 32), (6, 0), (7, args[7].repeat(2)), (8, args[8][:1]),
                    (8, args[8].float()), (9, args[9][:3]), (9, args[9][:, :0]), (9, torch.zeros(T, 9, dtype=torch.int32, device="cuda")), (9, args[9].flatten()),
                    (10, 0), (10, 1 << 31), (11, 0.0), (11, -1.0), (11, math.nan)]:
        with pytest.raises((ValueError, TypeError, kernels.KernelError)):
            kernels.tree_attention(*args[:at], bad, *args[at + 1:])
    for out in (torch.empty(T, 255, device="cuda"), torch.empty(T, 256), torch.empty(T, 256, device="cuda").bfloat16(), args[0][:, :256],
                args[4].flatten()[:T * 256].view(T, 256)):
        with pytest.raises((ValueError, TypeError, kernels.KernelError)):
            kernels.tree_attention(*args, out=out)
    none = kernels.tree_attention(args[0][:0], *args[1:9], args[9][:0], *args[10:])
    assert none.shape == (0, 256)
    kernels.check_status()


# ---- verification ---------------------------------------------------------------------------------------------------

def verify(c, most, probs=None, draft=None):
    up = lambda t: None if t is None else t.cuda()
    got = kernels.verify_drafts(up(c["probs"]) if probs is None else probs, up(c["tokens"]), up(c["parents"]), ints(c["row0"]), up(c["draws"]), most,
                                up(c["draft"]) if draft is None else draft)
    return tuple(t.tolist() for t in got)


@pytest.mark.parametrize("draft", [False, True], ids=["looked up", "drawn"])
@pytest.mark.parametrize("sizes,V,shape", [
    ([1], 1, "tree"), ([1, 1], 5, "tree"), ([4], 2, "tree"), ([6, 1, 9], 30, "tree"), ([8, 3], 1000, "chain"), ([40] * 5, 50, "tree"),
    ([12] * 20, 8193, "tree"), ([5] * 3, 32003, "chain"), ([64, 2, 33], 999, "tree"), ([300], 64, "tree"), ([7] * 3, 151936, "tree"), ([1024], 33, "tree"),
])
def test_verification(sizes, V, shape, draft):
    for seed in range(4):
        c = make_verify(sizes, V, draft, seed=seed, shape=shape, near=0.3 + seed)
        most = max(1, max(sizes) - 1)
        want = plain_verify(c["probs"], c["tokens"], c["parents"].tolist(), c["row0"], c["draws"], most, c["draft"])
        assert verify(c, most) == want
    kernels.check_status()


@pytest.mark.parametrize("draft", [False, True], ids=["looked up", "drawn"])
def test_siblings_of_one_token_and_bounds_on_what_is_accepted(draft):
    for seed in range(20):
        c = make_verify([24, 9], 6, draft, seed=seed, near=2.0)         # six tokens: siblings meet
        for most in (1, 2, 23):
            want = plain_verify(c["probs"], c["tokens"], c["parents"].tolist(), c["row0"], c["draws"], most, c["draft"])
            assert verify(c, most) == want, (seed, most)
    kernels.check_status()


def test_draws_at_their_ends_and_tokens_that_may_not_come():
    V = 5000
    c = make_verify([4, 4, 4], V, False, seed=1)
    c["probs"][:, 100:4000] = 0.0
    c["probs"][:, 4990:] = 0.0
    for u in (0.0, 1.0 - 2.0 ** -24, 0.5):
        c["draws"][:] = u
        c["tokens"][:] = torch.tensor([0, 200, 4995, 7] * 3)
        want = plain_verify(c["probs"], c["tokens"], c["parents"].tolist(), c["row0"], c["draws"], 3)
        got = verify(c, 3)
        assert got == want
        for said in got[2]:
            assert all(t < 0 or t < 100 or 4000 <= t < 4990 for t in said)
    kernels.check_status()


def test_one_certain_token():
    V = 30000
    c = make_verify([3, 3], V, False, seed=2, shape="chain")
    c["probs"].zero_()
    c["probs"][:, 29999] = 1.0
    c["tokens"][:] = 29999
    c["draws"][:] = 0.999
    assert verify(c, 2) == ([2, 2], [[1, 2], [1, 2]], [[29999] * 3, [29999] * 3])
    kernels.check_status()


def test_a_draft_that_is_the_target_leaves_nothing_to_take_off():
    """A token refused although the two distributions are one can only come of a draw of 1: the target's own row is then drawn from."""
    c = make_verify([2, 2, 2], 700, True, seed=3)
    up = torch.tensor([0, 0, 2, 2, 4, 4])
    c["draft"] = c["probs"][up].clone()
    c["draws"][:] = torch.tensor([0.3, 1.0, 0.6, 0.2, 0.99, 1.0])
    want = plain_verify(c["probs"], c["tokens"], c["parents"].tolist(), c["row0"], c["draws"], 1, c["draft"])
    assert want[0] == [0, 1, 0]
    assert verify(c, 1) == want
    kernels.check_status()


def test_rows_that_lie_apart():
    c = make_verify([6, 5], 1003, True, seed=8)
    want = plain_verify(c["probs"], c["tokens"], c["parents"].tolist(), c["row0"], c["draws"], 5, c["draft"])
    wide = torch.full((11, 3005), math.nan, device="cuda")
    wide[:, 5:1008], wide[:, 2000:3003] = c["probs"].cuda(), c["draft"].cuda()
    assert verify(c, 5, probs=wide[:, 5:1008], draft=wide[:, 2000:3003]) == want
    kernels.check_status()


def test_distribution_of_what_is_said():
    """40,000 requests of one tree: the first token comes as often as the target has it.  Each count is within 5 standard deviations."""
    V, n = 7, 40000
    for draft in (False, True):
        one = make_verify([4], V, draft, seed=11, near=1.0)
        g = torch.Generator().manual_seed(5)
        tokens = one["tokens"].repeat(n)
        if draft:
            tokens = torch.multinomial(one["draft"].repeat(1, 1), n, replacement=True, generator=g).t().reshape(-1).int()
        c = {"probs": one["probs"].repeat(n, 1), "draft": one["draft"].repeat(n, 1) if draft else None, "tokens": tokens,
             "parents": torch.tensor([-1, 0, 0, 0], dtype=torch.int32).repeat(n), "row0": list(range(0, 4 * n + 1, 4)), "draws": torch.rand(4 * n, generator=g)}
        if draft:       # siblings are drawn from one distribution
            c["draft"] = one["draft"][1:2].repeat(4 * n, 1)
            c["tokens"] = torch.multinomial(one["draft"][1:2].repeat(4 * n, 1), 1, generator=g)[:, 0].int()
        said = verify(c, 3)[2]
        counts = torch.bincount(torch.tensor([s[0] for s in said]), minlength=V).double()
        p = one["probs"][0].double() / one["probs"][0].double().sum()
        assert bool(((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all()), (draft, counts / n, p)


def test_trees_and_rows_that_make_no_sense_are_reported():
    for what in ("parent", "token", "row0", "empty", "zeros"):
        c = make_verify([5, 5], 40, False, seed=4, shape="chain")
        c["draws"][:] = 0.0
        if what == "parent":
            c["parents"][7] = 4
        if what == "token":
            c["tokens"][2] = 40
        if what == "row0":
            c["row0"] = [0, 5, 12]
        if what == "empty":
            c["row0"] = [0, 5, 5]
        if what == "zeros":
            c["probs"][4] = math.nan
        accepted, path, said = verify(c, 4)
        if what == "parent":
            assert accepted == [4, 1] and path[1] == [1, -1, -1, -1]
        if what == "token":
            assert accepted == [1, 4]
        if what == "zeros":
            assert accepted == [4, 4] and said[0][4] == -1
        if what == "empty":
            assert accepted == [4, 0] and path[1] == [-1] * 4 and said[1] == [-1] * 5
        with pytest.raises(kernels.KernelError, match="tree of drafted"):
            kernels.check_status()
    kernels.check_status()


def test_refusals_of_verification():
    c = make_verify([4], 20, True, seed=0)
    args = [c["probs"].cuda(), c["tokens"].cuda(), c["parents"].cuda(), ints(c["row0"]), c["draws"].cuda(), 3, c["draft"].cuda()]
    kernels.verify_drafts(*args)
    for at, bad in [(0, args[0].cpu()), (0, args[0].double()), (0, args[0].t()), (0, args[0][:, :0]), (0, args[0][0]), (1, args[1].long()), (1, args[1][:3]),
                    (1, args[1].cpu()), (2, args[2].repeat(2)), (3, args[3].view(1, 2)), (3, args[3][:0]), (4, args[4].double()), (4, args[4].cpu()),
                    (4, args[4][::2]), (5, 0), (5, 1025), (6, args[6][:, :19]), (6, args[6].expand(4, 20)[:, :1].expand(4, 20)), (6, args[6].cpu())]:
        with pytest.raises((ValueError, TypeError, kernels.KernelError)):
            kernels.verify_drafts(*args[:at], bad, *args[at + 1:])
    accepted, path, said = kernels.verify_drafts(*args[:3], args[3][:1], *args[4:])
    assert accepted.shape == (0,) and path.shape == (0, 3) and said.shape == (0, 4)
    kernels.check_status()


# ---- rows and pages ---------------------------------------------------------------------------------------------------

def rising(rnd, n, most):
    return sorted(rnd.sample(range(1, most + 1), n))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8], ids=["f32", "bf16", "u8"])
@pytest.mark.parametrize("layers,heads,width,ps,sizes,lengths", [
    (1, 1, 16, 16, [2], [0]), (3, 2, 32, 16, [9, 30, 2], [15, 100, 7]), (5, 4, 128, 64, [200], [60]), (2, 3, 10, 7, [20, 20], [3, 50]), (28, 4, 64, 32, [8] * 40, [31] * 40),
    (2, 1, 18, 16, [300], [5]),
])
def test_kept_rows_move_up(layers, heads, width, ps, sizes, lengths, dtype):
    rnd, g = random.Random(width), torch.Generator().manual_seed(width)
    table, n = block_tables([a + b for a, b in zip(sizes, lengths)], ps, rnd)
    most = max(sizes) - 1
    paths = [rising(rnd, rnd.randint(0, s - 1), s - 1) for s in sizes]
    paths[0] = rising(rnd, sizes[0] - 1 if sizes[0] < 100 else 150, sizes[0] - 1)
    accepted = [len(p) for p in paths]
    path = [p + [-1] * (most - len(p)) for p in paths]
    pages = torch.randint(0, 200, (layers, n, 2, heads, ps, width), generator=g).to(dtype)
    want = plain_compact(pages.flatten(2, 3), table, lengths, path, accepted).view(pages.shape)
    got = pages.cuda()
    kernels.compact_cache(got, table.cuda(), ints(lengths), ints(path), ints(accepted))
    assert torch.equal(got.cpu(), want)
    # one layer by itself, and rows of any width
    got = pages.cuda()
    for li in range(layers):
        kernels.compact_cache(got[li], table.cuda(), ints(lengths), ints(path), ints(accepted))
    assert torch.equal(got.cpu(), want)
    got = pages[:, :, 0, 0].contiguous().cuda()
    kernels.compact_cache(got, table.cuda(), ints(lengths), ints(path), ints(accepted))
    assert torch.equal(got.cpu(), want[:, :, 0, 0])
    kernels.check_status()


def test_paths_that_make_no_sense_move_nothing():
    table, n = block_tables([40, 40], 16, random.Random(0))
    pages = torch.randn(2, n, 2, 1, 16, 32, device="cuda")
    before = pages.clone()
    for path, accepted, length in [([2, 2], 2, 3), ([3, 1], 2, 3), ([0, 5], 2, 3), ([2, 3], 3, 3), ([2, 3], -1, 3), ([2, 10 ** 9], 1, -4), ([-1, -1], 1, 3)]:
        kernels.compact_cache(pages, table.cuda(), ints([3, length]), ints([[-1, -1], path]), ints([0, accepted]))
        assert torch.equal(pages, before)
        with pytest.raises(kernels.KernelError, match="copy of cache rows"):
            kernels.check_status()
    # a page outside the pool: that row stays, the others move
    bad = table.clone()
    bad[1, 1] = 10 ** 6
    kernels.compact_cache(pages, bad.cuda(), ints([3, 3]), ints([[-1, -1], [5, 20]]), ints([0, 2]))
    row = lambda t, at: t[:, table[1, at // 16].long(), :, :, at % 16]
    assert torch.equal(row(pages, 4), row(before, 8)) and torch.equal(row(pages, 5), row(before, 5))
    with pytest.raises(kernels.KernelError, match="copy of cache rows"):
        kernels.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8], ids=["f32", "bf16", "u8"])
@pytest.mark.parametrize("shape", [(1, 5, 2, 1, 16, 16), (3, 40, 2, 4, 64, 128), (2, 9, 2, 3, 7, 10), (4, 30, 16, 72), (6, 3, 1), (12, 2, 2, 16, 6)])
def test_copied_pages(shape, dtype):
    if shape[-1] % 2 and dtype == torch.uint8:
        return
    rnd, g = random.Random(len(shape)), torch.Generator().manual_seed(3)
    pages = torch.randint(0, 200, shape, generator=g).to(dtype)
    at = 1 if len(shape) in (4, 6) else 0
    order = rnd.sample(range(shape[at]), shape[at])
    n, ps = shape[at] // 2, shape[-2]
    src, dst = order[:n], order[n:2 * n]
    for rows in (None, [rnd.randint(0, ps) for _ in range(n)]):
        want = pages.clone()
        view, new = (want, pages) if at else (want[None], pages[None])
        for i, (a, b) in enumerate(zip(src, dst)):
            k = ps if rows is None else rows[i]
            view[:, b, ..., :k, :] = new[:, a, ..., :k, :]
        got = pages.cuda()
        kernels.copy_pages(got, ints(src), ints(dst), None if rows is None else ints(rows))
        assert torch.equal(got.cpu(), want)
    kernels.check_status()


def test_more_copies_and_requests_than_a_dimension_of_a_grid():
    n = 70000
    pages = torch.arange(2 * n * 8, dtype=torch.int32, device="cuda").view(2 * n, 2, 4)
    src, dst = torch.randperm(n, generator=torch.Generator().manual_seed(0)).int(), torch.arange(n, 2 * n, dtype=torch.int32)
    want = pages.clone()
    want[n:] = want[:n][src.long().cuda()]
    kernels.copy_pages(pages, src.cuda(), dst.cuda())
    assert torch.equal(pages, want)
    # the second row of every request's only page takes the place of the first behind its root's: page_size 3, path [2]
    rows = torch.arange(n * 6, device="cuda").to(torch.int16).view(n, 3, 2)
    want = rows.clone()
    kept = torch.zeros(n, dtype=torch.int32)
    kept[[0, 65535, 65536, n - 1]] = 1
    want[[0, 65535, 65536, n - 1], 1] = want[[0, 65535, 65536, n - 1], 2]
    kernels.compact_cache(rows, torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1), torch.zeros(n, dtype=torch.int32, device="cuda"),
                          torch.full((n, 1), 2, dtype=torch.int32, device="cuda"), kept.cuda())
    assert torch.equal(rows, want)
    kernels.check_status()


def test_layers_that_lie_apart_and_pages_onto_themselves():
    whole = torch.randn(6, 8, 2, 2, 16, 32, device="cuda")
    before = whole.clone()
    part = whole[1::2]
    kernels.copy_pages(part, ints([0, 3]), ints([1, 3]))
    assert torch.equal(whole[0::2], before[0::2])
    before[1::2, 1] = before[1::2, 0]
    assert torch.equal(whole, before)
    kernels.check_status()


def test_entries_outside_the_pool_are_left_out():
    pages = torch.randn(2, 6, 2, 1, 16, 32, device="cuda")
    before = pages.clone()
    for src, dst, rows in [([-1], [2], None), ([6], [2], None), ([1], [-1], None), ([1], [6], None), ([1], [2], [17]), ([1], [2], [-1])]:
        kernels.copy_pages(pages, ints(src), ints(dst), None if rows is None else ints(rows))
        assert torch.equal(pages, before)
        with pytest.raises(kernels.KernelError, match="copy of cache rows"):
            kernels.check_status()
    kernels.check_status()


def test_refusals_of_copies():
    pages = torch.zeros(2, 6, 2, 1, 16, 32, device="cuda")
    one = ints([1])
    for args in [(pages.cpu(), one, ints([2])), (pages.transpose(1, 2), one, ints([2])), (pages[0, 0, 0, 0], one, ints([2])), (pages, one.long(), ints([2])),
                 (pages, one, ints([2, 3])), (pages, one, ints([2]), ints([1, 2])), (pages, one.cpu(), ints([2])), (pages[:, :0], one, ints([2])),
                 (torch.zeros(2, 6, 16, 3, device="cuda", dtype=torch.uint8), one, ints([2])), (pages, ints([[1]]), ints([[2]]))]:
        with pytest.raises((ValueError, TypeError, kernels.KernelError)):
            kernels.copy_pages(*args)
    table, path = ints([[0, 1]]), ints([[3]])
    good = [pages, table, one, path, one]
    kernels.compact_cache(*good)
    for at, bad in [(0, pages.cpu()), (0, pages[..., ::2]), (1, table.long()), (1, table[0]), (1, table[:, :0]), (2, ints([1, 2])), (2, one.cpu()), (3, path[0]),
                    (3, ints([[3], [4]])), (4, ints([1, 1])), (4, one.float())]:
        with pytest.raises((ValueError, TypeError, kernels.KernelError)):
            kernels.compact_cache(*good[:at], bad, *good[at + 1:])
    kernels.copy_pages(pages, ints([]), ints([]))
    kernels.check_status()
