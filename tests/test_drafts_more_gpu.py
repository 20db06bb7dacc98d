"""Trees of drafted tokens where a call goes from one piece of work to the next, or its operands do not fit, against plain
forms in 64 bits."""

import random

import pytest
import torch

from ninfer_amd_mi50_b200 import kernels
from ninfer_amd_mi50_b200.kernels import drafts
from plain_drafts import make_attention, make_verify, plain_attention, plain_verify
from test_drafts_gpu import attend, near, verify

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


def without_missing_pages(c, heads, page_size, pool):
    """What is left of a step (plain_attention's operands, pages of one row) when nobody sees keys whose page is not there."""
    lengths, table, mask, rows = [], [], c["mask"].clone(), [torch.zeros(2, heads[1], 1, heads[2])]
    for s, (lo, hi) in enumerate(zip(c["row0"], c["row0"][1:])):
        at, held = [], 0
        for j in range(c["lengths"][s] + hi - lo):
            page = int(c["table"][s, j // page_size]) if j // page_size < c["table"].shape[1] else -1
            there = 0 <= page < pool
            if there:
                rows.append(c["pages"][page, :, :, j % page_size, None])
            if j < c["lengths"][s]:
                held += there
            elif not there:                                    # a node that nobody sees
                k = j - c["lengths"][s]
                mask[lo:hi, k // 32] &= ~(1 << k % 32) if k % 32 < 31 else 0x7fffffff
            if there or j >= c["lengths"][s]:
                at.append(len(rows) - 1 if there else 0)
        lengths.append(held)
        table.append(at)
    width = max(1, max(len(t) for t in table))
    return torch.stack(rows), torch.tensor([t + [-1] * (width - len(t)) for t in table], dtype=torch.int32), lengths, mask


@pytest.mark.parametrize("form,dtype,heads,page_size,sizes,lengths", [
    ("auto", torch.float32, (4, 2, 64), 16, [9, 6, 4], [300, 90, 40]),
    (0, torch.bfloat16, (6, 2, 48), 7, [9, 6, 4], [100, 90, 40]),
    (1, torch.bfloat16, (4, 2, 64), 16, [9, 6, 4], [300, 90, 40]),
    (1, torch.bfloat16, (24, 1, 64), 32, [17, 2, 40], [700, 200, 129]),
    (1, torch.bfloat16, (16, 2, 128), 64, [40, 9, 33], [900, 30, 500]),
    (1, torch.bfloat16, (8, 2, 128), 128, [70, 9, 33], [900, 30, 500]),
    (1, torch.bfloat16, (4, 4, 128), 16, [9] * 30, [300, 500, 700] * 10),
    (2, torch.bfloat16, (4, 2, 64), 16, [9, 6, 4], [300, 90, 40]),
    (2, torch.bfloat16, (24, 1, 64), 32, [17, 2, 40], [700, 200, 129]),
    (2, torch.bfloat16, (4, 4, 128), 64, [3, 4, 1], [900, 30, 500]),
    (2, torch.bfloat16, (16, 2, 128), 128, [40, 9, 33], [900, 30, 500]),
    (2, torch.bfloat16, (4, 2, 128), 48, [9, 6, 4], [900, 30, 500]),
], ids=lambda v: f"{len(v)} requests" if isinstance(v, list) else str(v).replace("torch.", ""))
def test_keys_of_missing_pages_are_not_seen(form, dtype, heads, page_size, sizes, lengths, asked):
    """Whatever shared memory still holds there: a call whose keys and values are NaN comes before."""
    asked(form)
    for what in ("some", "first", "last", "all of a request", "beyond the table"):
        c = make_attention(sizes, lengths, heads, page_size, seed=7)
        c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
        pool, table = c["pages"].shape[0], c["table"]
        attend({**c, "pages": torch.full_like(c["pages"], float("nan"))}, heads, page_size, dtype, 0.2)
        kernels.check_status()
        if what == "some":
            gone = torch.rand(table.shape, generator=torch.Generator().manual_seed(3)) < 0.3
            table[gone] = torch.tensor([-1, pool, 10 ** 6, -2 ** 31], dtype=torch.int32).repeat(table.numel())[:int(gone.sum())]
        if what == "first":
            table[:, 0] = -1
        if what == "last":
            for s, n in enumerate(sizes):
                table[s, (lengths[s] + n - 1) // page_size] = pool
        if what == "all of a request":
            table[0] = -1
        if what == "beyond the table":
            c["table"] = table[:, :max(1, table.shape[1] // 2)].contiguous()
        pages, rows, held, mask = without_missing_pages(c, heads, page_size, pool)
        want, weight, size = plain_attention(c["qkv"], *heads, pages, rows, 1, held, c["row0"], mask, 0.2)
        got = attend(c, heads, page_size, dtype, 0.2)
        assert form == "auto" or form_of(c, heads, page_size) == form
        near(got, want, weight, size, c["longest"], dtype, heads[2])
        assert torch.equal(got, attend(c, heads, page_size, dtype, 0.2))
        with pytest.raises(kernels.KernelError, match="tree of drafted"):
            kernels.check_status()


@pytest.mark.parametrize("form", ["auto", 0, 1, 2])
def test_rows_and_lengths_outside_their_bounds_count_as_if_they_ended_there(form, asked):
    asked(form)
    heads, dtype = (4, 2, 64), torch.float32 if form == "auto" else torch.bfloat16
    for what in ("context", "row0", "length"):
        c = make_attention([4, 6], [40, 90], heads, 16, seed=6)
        c["qkv"], c["pages"] = c["qkv"].to(dtype).float(), c["pages"].to(dtype).float()
        plain = {**c}
        if what == "context":                                  # the second request's keys end there, its nodes' with them
            c["longest"] = 64
            plain["lengths"], plain["mask"] = [40, 64], c["mask"].clone()
            plain["mask"][4:] = 0
        if what == "row0":
            c["row0"], plain["row0"] = [0, 4, 99], [0, 4, 10]
        if what == "length":
            c["lengths"], plain["lengths"] = [-3, 90], [0, 90]
        want, weight, size = plain_attention(plain["qkv"], *heads, plain["pages"], plain["table"], 16, plain["lengths"], plain["row0"], plain["mask"], 0.2)
        near(attend(c, heads, 16, dtype, 0.2), want, weight, size, c["longest"], dtype, heads[2])
        with pytest.raises(kernels.KernelError, match="tree of drafted"):
            kernels.check_status()


@pytest.mark.parametrize("draft", [False, True], ids=["looked up", "drawn"])
def test_probabilities_that_are_no_positive_numbers_count_as_none(draft):
    """In the target's rows and in the draft's, at drafted tokens too."""
    for seed in range(30):
        c = make_verify([12, 5, 30], 40, draft, seed=seed, near=1.0)
        g = torch.Generator().manual_seed(seed)
        odd = torch.tensor([float("nan"), -0.25, -float("inf"), -0.0, -1e30])
        plain = dict(c)
        for name in ("probs", "draft") if draft else ("probs",):
            at = torch.rand(c[name].shape, generator=g) < 0.3
            at[:, ::7] = False                                 # (something is left of every row)
            c[name] = torch.where(at, odd[torch.randint(len(odd), at.shape, generator=g)], c[name])
            plain[name] = torch.where(at, torch.zeros(()), c[name])
        want = plain_verify(plain["probs"], c["tokens"], c["parents"].tolist(), c["row0"], c["draws"], 29, plain["draft"])
        assert verify(c, 29) == want, seed
    kernels.check_status()


@pytest.mark.parametrize("draft", [False, True], ids=["looked up", "drawn"])
@pytest.mark.parametrize("at", [0, 20000, 29999])
def test_a_row_that_holds_something_infinite_says_nothing(at, draft):
    c = make_verify([4, 3], 30000, draft, seed=2, shape="chain")
    c["draws"][:] = torch.tensor([0.5, 0.0, 0.0, 0.0, 0.3, 0.0, 0.0])
    c["probs"][3, at] = float("inf")
    accepted, path, said = verify(c, 3)
    assert accepted == [3, 2] and path == [[1, 2, 3], [1, 2, -1]] and said[0] == c["tokens"][1:4].tolist() + [-1]
    assert 0 <= said[1][2] < 30000
    with pytest.raises(kernels.KernelError, match="tree of drafted"):
        kernels.check_status()


@pytest.mark.parametrize("form", [0, 1, 2])
def test_scales_that_float32_does_not_hold_are_refused(form, asked):
    asked(form)
    heads = (4, 2, 64)
    c = make_attention([9, 4], [40, 130], heads, 16, seed=1)
    c["qkv"], c["pages"] = c["qkv"].bfloat16().float(), c["pages"].bfloat16().float()
    for bad in (1e-50, 2.0 ** -127, 2.0 ** 127, 1e39, float("inf"), -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            attend(c, heads, 16, torch.bfloat16, bad)
    # the least one: every key that is seen counts as much
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], 16, c["lengths"], c["row0"], c["mask"], 2.0 ** -126)
    near(attend(c, heads, 16, torch.bfloat16, 2.0 ** -126), want, weight, size, c["longest"], torch.bfloat16, 64)
    kernels.check_status()


@pytest.mark.parametrize("form", [0, 1, 2])
def test_which_sizes_each_form_takes(form, asked):
    """A form that is asked for serves every size that it takes, and another one the rest."""
    asked(form)
    for dtype in (torch.bfloat16, torch.float32):
        for heads, page_size in [((4, 2, 64), 16), ((4, 2, 64), 32), ((4, 2, 128), 64), ((1, 1, 128), 128), ((28, 4, 128), 64), ((4, 2, 64), 48), ((2, 2, 128), 96),
                                 ((4, 2, 128), 256), ((4, 2, 64), 8), ((4, 2, 64), 7), ((6, 2, 48), 16), ((4, 1, 256), 64), ((3, 3, 80), 64)]:
            c = make_attention([3], [20], heads, page_size, seed=1)
            attend(c, heads, page_size, dtype, 0.1)
            whole = dtype == torch.bfloat16 and heads[2] in (64, 128) and page_size % 16 == 0
            tc = whole and page_size in (16, 32, 64, 128)
            key = next(k for k in reversed(drafts._plans) if k[2:6] == (*heads, page_size) and k[-1] == form and k[9] == (dtype == torch.bfloat16))
            # (one request of three nodes: what form 1 does not take and whatever is little goes to form 2, the rest to CUDA cores)
            assert drafts._plans[key][0] & 3 == (0 if form == 0 or not whole else (1 if form == 1 and tc else 2)), (dtype, heads, page_size)
    kernels.check_status()


@pytest.mark.parametrize("form", [1, 2])
@pytest.mark.parametrize("heads,most,page_size", [((24, 2, 128), 30, 64), ((8, 8, 64), 40, 16), ((5, 1, 128), 64, 128)])
def test_every_row_of_many_requests(heads, most, page_size, form, asked):
    """More work than there are SMs, in items of one tile of rows and of two, each row against the plain form."""
    asked(form)
    rnd = random.Random(most)
    sizes = [rnd.randint(0 if s else 1, most) for s in range(30)]
    lengths = [rnd.choice([0, 1, 127, 128, 129, rnd.randint(0, 600), rnd.randint(0, 300)]) for _ in sizes]
    c = make_attention(sizes, lengths, heads, page_size, seed=most, words=2)
    c["qkv"], c["pages"] = c["qkv"].bfloat16().float(), c["pages"].bfloat16().float()
    want, weight, size = plain_attention(c["qkv"], *heads, c["pages"], c["table"], page_size, c["lengths"], c["row0"], c["mask"], 0.1)
    got = attend(c, heads, page_size, torch.bfloat16, 0.1)
    assert form_of(c, heads, page_size) == form
    near(got, want, weight, size, c["longest"], torch.bfloat16, heads[2])
    kernels.check_status()
