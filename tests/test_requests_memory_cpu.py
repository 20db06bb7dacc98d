"""What the host knows about the memory of a call's rows, without a GPU."""

import torch

from ninfer_amd_mi50_b200.kernels.requests import _clash, _overlap, _rows_apart


def test_rows_apart():
    flat = torch.empty(1 << 33, device="meta")
    at = lambda *strides, shape=(3, 5): _rows_apart(flat.as_strided(shape, strides), *shape)
    assert at(5, 1) == 5 and at(9, 1) == 9 and at((1 << 31) - 1, 1) == (1 << 31) - 1
    # a step of 2^32 + 5 is 5 in 32 bits: rows that are not asked for
    assert at(1 << 31, 1) == -1 and at((1 << 32) + 5, 1) == -1
    assert at(4, 1) == -1 and at(0, 1) == -1 and at(5, 2) == -1
    assert at((1 << 32) + 5, 1, shape=(1, 5)) == 5 and at(7, 3, shape=(3, 1)) == 7


def test_shared_rows_by_trying_every_place():
    def shares(p, a, q, b, R, V):
        one = {p + 4 * (r * a + i) for r in range(R) for i in range(V)}
        other = {q + 4 * (r * b + i) for r in range(R) for i in range(V)}
        return bool(one & other)

    for R, V in ((1, 3), (2, 3), (3, 4), (4, 1)):
        for a in range(V, 2 * V + 4):
            for b in range(V, 2 * V + 4):
                for q in range(-40, 41):
                    got = _clash(400, a, 400 + 4 * q, b, R, V)
                    if q == 0 and (a == b or R == 1):
                        assert not got
                    elif shares(400, a, 400 + 4 * q, b, R, V):
                        assert got
                    elif a == b:                     # (rows at other distances, one among the other, are refused unseen)
                        assert not got, (R, V, a, q)


def test_overlap():
    t = torch.zeros(64)
    assert _overlap(t[:32], t[31:40]) and _overlap(t, t) and not _overlap(t[:32], t[32:]) and not _overlap(t[32:], t[:32])
