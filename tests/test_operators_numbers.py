"""The handle-less operators' numbers: what the library could only take in
part, or not at all, is refused with ValueError."""
from decimal import Decimal
from fractions import Fraction

import numpy as np
import pytest
import torch

from gotransformers_b200 import moe, operators


@pytest.mark.parametrize("seed,stream,offset", [
    (0, 0, 1 << 63), (0, 0, 1 << 64), (0, 0, (1 << 64) + 5), (0, 0, -(1 << 63) - 1),
    (1.0, 0, 0), (0, "1", 0), (0, 0, 2.0), (None, 0, 0),
])
def test_generator_numbers_that_are_refused(seed, stream, offset):
    with pytest.raises(ValueError):
        operators._generator(seed, stream, offset)


def test_generator_numbers():
    word = (1 << 64) - 1
    assert operators._generator(word, word, (1 << 63) - 1) == [word, word, (1 << 63) - 1]
    assert operators._generator(-1, -(1 << 63), -1) == [word, 1 << 63, -1]  # the library refuses the offset
    assert operators._generator((1 << 64) + 3, 1 << 70, 0) == [3, 0, 0]
    got = operators._generator(np.int64(7), np.uint64(word), np.int32(9))
    assert got == [7, word, 9] and all(type(v) is int for v in got)


def test_real_numbers():
    for v in (0.5, 1, np.float32(0.5), np.float64(0.25), True, torch.tensor(0.5), Decimal("0.25"), Fraction(1, 8)):
        assert operators._number("rate", v) == float(v) and type(operators._number("rate", v)) is float
    for v in (None, "0.5", b"0.5", 1j, [0.5], torch.ones(2)):
        with pytest.raises(ValueError):
            operators._number("rate", v)


@pytest.mark.gpu
def test_offsets_past_the_librarys_range_make_no_decisions():
    """2^64 was seen as 0: the first elements' decisions, without a word."""
    x = torch.ones(64, device="cuda")
    calls = [
        lambda: moe.dropout(x, 0.5, 1, 0, 1 << 64),
        lambda: moe.dropout_backward(x, 0.5, 1, 0, 1 << 64),
        lambda: moe.dropout(x, "half", 1),
        lambda: moe.layer_norm(x.view(2, 32), epsilon="small"),
    ]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    # numpy's numbers are numbers
    assert torch.equal(moe.dropout(x, np.float64(0.5), np.int64(3), np.int32(1)), moe.dropout(x, 0.5, 3, 1))
