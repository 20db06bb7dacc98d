"""What the host knows about the memory of a call's rows, without a GPU."""

import torch

from ninfer_amd_mi50_b200.kernels.requests import _rows_apart


def test_rows_apart():
    flat = torch.empty(1 << 33, device="meta")
    at = lambda *strides, shape=(3, 5): _rows_apart(flat.as_strided(shape, strides), *shape)
    assert at(5, 1) == 5 and at(9, 1) == 9 and at((1 << 31) - 1, 1) == (1 << 31) - 1
    # a step of 2^32 + 5 is 5 in 32 bits: rows that are not asked for
    assert at(1 << 31, 1) == -1 and at((1 << 32) + 5, 1) == -1
    assert at(4, 1) == -1 and at(0, 1) == -1 and at(5, 2) == -1
    assert at((1 << 32) + 5, 1, shape=(1, 5)) == 5 and at(7, 3, shape=(3, 1)) == 7
