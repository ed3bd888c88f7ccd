"""Operands of the block operators as programs hold them: results beside their
operands in one buffer, single tokens and views that start anywhere."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import fused_linear
from oracle.block import linear_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16


def _randn(*shape, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(BF16)


@pytest.mark.parametrize("m", [4, 300])
def test_a_result_beside_its_operand_and_over_it(m):
    k, n = 64, 48
    w, buffer = _randn(n, k, seed=1, scale=0.1), _randn(m, k + n, seed=2)
    x, out = buffer[:, :k], buffer[:, k:]
    want, bound = linear_reference(x.clone(), w)
    assert fused_linear(x, w, out=out).data_ptr() == out.data_ptr()
    assert ((out.double() - want).abs() <= bound).all()
    square = _randn(k, k, seed=3)
    for other in (buffer[:, :k], buffer[:, 16 : 16 + k]):
        with pytest.raises(ValueError, match="overlap"):
            fused_linear(x, square, out=other)
    with pytest.raises(ValueError, match="overlap"):
        fused_linear(_randn(k, k, seed=4), square, out=square)
