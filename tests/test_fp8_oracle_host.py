"""What the 8-bit layers' results are held to refuses wrong ones: values, scales and NaN
planted in the pairs that oracle.fp8.check_groups is given."""

from __future__ import annotations

import pytest
import torch

from oracle.fp8 import check_groups, quantize_reference

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture
def pair():
    """(e4m3 bytes, e8m0 bytes, values) of a right rounding, and room for none but half a step."""
    y = torch.randn((6, 272), generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    q, byte = quantize_reference(y)
    return q.to(E4M3).view(torch.uint8), byte.to(torch.uint8), y


def _check(q, byte, y):
    check_groups(q.view(E4M3), byte.view(E8M0), y, torch.zeros_like(y))


def test_a_right_pair_is_taken(pair):
    _check(*pair)


@pytest.mark.parametrize("row, column", [(0, 0), (3, 130), (5, 271)])
@pytest.mark.parametrize("nan", [0x7F, 0xFF])
def test_a_value_that_is_nan_is_refused(pair, nan, row, column):
    q, byte, y = pair
    q[row, column] = nan
    with pytest.raises(AssertionError):
        _check(q, byte, y)


def test_nothing_but_nan_is_refused(pair):
    q, byte, y = pair
    with pytest.raises(AssertionError):
        _check(torch.full_like(q, 0x7F), byte, y)


def test_a_value_two_steps_away_and_another_scale_are_refused(pair):
    q, byte, y = pair
    j = int(y[2].abs().argmax())
    for wrong_q, wrong_byte in ((q.clone(), byte), (q, byte.clone())):
        if wrong_q is not q:
            wrong_q[2, j] -= 2
        else:
            wrong_byte[2, j // 128] += 1
        with pytest.raises(AssertionError):
            _check(wrong_q, wrong_byte, y)


def test_a_reference_that_is_not_finite_is_refused(pair):
    # it would hold nothing to anything
    q, byte, y = pair
    y[1, 5] = float("nan")
    with pytest.raises(AssertionError):
        _check(q, byte, y)
