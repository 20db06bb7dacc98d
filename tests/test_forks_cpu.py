"""Requests forked, and trees of drafted tokens, on the host: pages with several holders are neither lost nor freed while
somebody holds them, what a fork copies, and which trees and paths are refused."""

import random

import pytest
import torch

from ninfer_amd_mi50_b200.cache import CacheManager, OutOfPages, OutOfSlots, PagePool
from ninfer_amd_mi50_b200.engine.batch import BatchError, TreeEntry, tree_parents, tree_rows
from ninfer_amd_mi50_b200.parts.base import CacheSpec, StateSpec

FULL = CacheSpec("full", 2, 16)
WIN = CacheSpec("window", 2, 16, 40)


def manager(specs=(FULL, FULL), states=(None, None), pages=12, reqs=4, allocate=True):
    return CacheManager(list(specs), list(states), page_size=16, num_pages=pages, max_requests=reqs, max_context=256, allocate=allocate)


def fill(m, req, to, value):
    """Positions up to `to` of a request, as a step would: their entries hold `value` in every layer."""
    at = m.length(req)
    m.reserve(req, to)
    for g in m.groups:
        for pos in range(at, to):
            g.pages[:, m.block_table(g.index, req)[pos // 16], :, :, pos % 16] = value
    m.commit(req, to)


def held(m, req, group=0):
    """What a request reads of its first layer: one number a position, None where a window has passed."""
    g, t = m.groups[group], m.block_table(group, req)
    return [float(g.pages[0, t[p // 16], 0, 0, p % 16, 0]) if t[p // 16] >= 0 else None for p in range(m.length(req))]


def test_pool_with_several_holders():
    p = PagePool(3)
    a = p.take(2)
    p.share(a)
    p.share(a[:1])
    p.give_back(a)
    assert p.num_free == 1 and p.holders(a[0]) == 2 and p.holders(a[1]) == 1
    p.check()
    p.give_back(a)
    assert p.num_free == 2 and p.holders(a[1]) == 0
    with pytest.raises(AssertionError, match="freed twice"):
        p.give_back([a[1]])
    with pytest.raises(AssertionError, match="nobody holds"):
        p.share([a[1]])
    p.give_back([a[0]])
    assert p.num_free == 3
    p.check()


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 40, 64])
def test_a_fork_reads_the_same_and_goes_on_by_itself(length):
    m = manager()
    m.open("a")
    if length:
        fill(m, "a", length, 1.0)
    free = m.pages_free()[0]
    m.fork("a", "b")
    m.check()
    assert m.length("b") == length and held(m, "b") == [1.0] * length
    assert m.pages_free()[0] == free - (length % 16 > 0)             # the page filled in part alone was copied
    fill(m, "a", length + 20, 2.0)
    fill(m, "b", length + 3, 3.0)
    assert held(m, "a") == [1.0] * length + [2.0] * 20
    assert held(m, "b") == [1.0] * length + [3.0] * 3
    m.check()
    m.close("a")
    m.check()
    assert held(m, "b") == [1.0] * length + [3.0] * 3
    m.close("b")
    assert m.pages_free() == [12]
    m.check()


def test_a_fork_takes_states_along_and_window_pages_are_given_back_by_each():
    m = manager(specs=(FULL, WIN), states=(StateSpec((3,)), None), pages=20)
    m.open("a")
    fill(m, "a", 70, 1.0)
    m.state[0][m.slot("a")] = 5.0
    m.fork("a", "b")
    assert bool((m.state[0][m.slot("b")] == 5.0).all())
    m.state[0][m.slot("b")] = 6.0
    assert bool((m.state[0][m.slot("a")] == 5.0).all())
    assert held(m, "b", 1) == held(m, "a", 1) and None in held(m, "a", 1)
    fill(m, "a", 130, 2.0)
    m.check()
    assert held(m, "b", 1)[-40:] == [1.0] * 40                       # "a" has left pages that "b" still reads
    fill(m, "b", 90, 3.0)
    m.check()
    for r in ("a", "b"):
        m.close(r)
    assert m.pages_free() == [20, 20]
    m.check()


def test_a_fork_that_finds_no_room_changes_nothing():
    m = manager(pages=3, reqs=2)
    m.open("a")
    fill(m, "a", 40, 1.0)
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    assert not m.is_open("b") and m.pages_free() == [0]
    m.check()
    m.close("a")
    m.open("a")
    fill(m, "a", 32, 1.0)
    m.fork("a", "b")                                                 # (whole pages need no other)
    with pytest.raises(OutOfSlots):
        m.fork("a", "c")
    with pytest.raises(KeyError):
        m.fork("nobody", "c")
    m.close("b")
    with pytest.raises(KeyError):
        m.fork("a", "a")
    m.check()


def test_forks_in_any_order():
    for seed in range(20):
        rnd = random.Random(seed)
        m = manager(specs=(FULL, WIN, FULL), states=(None, None, None), pages=24, reqs=5)
        live, n = {}, 0
        for _ in range(120):
            what = rnd.choice(["open", "fork", "run", "run", "close", "tree"])
            req = rnd.choice(sorted(live)) if live else None
            try:
                if what == "open" or req is None:
                    m.open(f"r{n}")
                    live[f"r{n}"] = []
                    n += 1
                elif what == "fork":
                    m.fork(req, f"r{n}")
                    live[f"r{n}"] = list(live[req])
                    n += 1
                elif what == "run" and len(live[req]) < 200:
                    to, v = len(live[req]) + rnd.randint(1, 30), float(n + rnd.random())
                    fill(m, req, to, v)
                    live[req] += [torch.tensor(v).item()] * (to - len(live[req]))
                elif what == "tree" and len(live[req]) < 200:        # reserved, then left
                    m.reserve(req, len(live[req]) + rnd.randint(1, 40))
                    if rnd.random() < 0.5:
                        m.truncate(req)
                elif what == "close":
                    m.close(req)
                    del live[req]
            except (OutOfPages, OutOfSlots):
                pass
            m.check()
            for r, want in live.items():
                got = held(m, r)
                assert got == pytest.approx(want) and len(got) == len(want)
        for r in list(live):
            m.close(r)
        assert m.pages_free() == [24, 24]


def test_trees():
    rows = tree_rows([10, 0], [[-1, 0, 0, 1, 3], [-1]], torch.device("cpu"))
    assert rows.positions.tolist() == [10, 11, 11, 12, 13, 0]
    assert rows.mask.tolist() == [[1], [3], [5], [11], [27], [1]]
    chain = tree_rows([5], [[-1] + list(range(69))], torch.device("cpu"))
    assert chain.mask.shape == (70, 3) and chain.mask[69].tolist() == [-1, -1, 63] and chain.mask[31].tolist() == [-1, 0, 0]
    assert chain.positions.tolist() == list(range(5, 75))


def test_trees_that_are_none_are_refused():
    good = TreeEntry("r", [5, 6, 7, 8])
    assert tree_parents(good, 8) == [-1, 0, 1, 2]
    assert tree_parents(TreeEntry("r", [5, 6, 7], [9, 0, 0]), 8) == [-1, 0, 0]           # (the root's is not read)
    for tokens, parents in [([5, 6], [-1]), ([5, 6], [-1, 1]), ([5, 6], [-1, -1]), ([5, 6, 7], [-1, 2, 0]), ([5] * 9, None), ([5], [])]:
        if parents == []:
            assert tree_parents(TreeEntry("r", tokens, parents), 8) == [-1]
            continue
        with pytest.raises(BatchError):
            tree_parents(TreeEntry("r", tokens, parents), 8)
