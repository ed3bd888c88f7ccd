"""Operands of the block operators as programs hold them: results beside their
operands in one buffer, single tokens and views that start anywhere."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import flash_attn_func, fused_linear, select_key_blocks, sparse_attn_func
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


def _starting_anywhere(t):
    """t's values in a contiguous view that starts 2 bytes into a buffer."""
    buffer = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return buffer[1:].view(t.shape).copy_(t)


def _one_token(t):
    """t's values, one token, as a row of a buffer of rows of an odd length."""
    batch, _, heads, d = t.shape
    row = heads * d + 1
    view = torch.empty(3 * batch * row, dtype=t.dtype, device=t.device).as_strided(t.shape, (3 * batch * row, row, d, 1), row - 1)
    return view.copy_(t)


@pytest.mark.parametrize("S, move", [(1, _starting_anywhere), (77, _starting_anywhere), (600, _starting_anywhere), (1, _one_token)])
def test_attention_operands_that_start_anywhere(S, move):
    q, k, v = (_randn(1, S, 2, 128, seed=10 + i) for i in range(3))
    moved = [move(t) for t in (q, k, v)]
    index = torch.zeros((1, 2, -(-S // 256), 1), dtype=torch.int32, device=DEV)
    assert torch.equal(select_key_blocks(*moved[:2], 1), select_key_blocks(q, k, 1))
    for got, want in ((flash_attn_func(*moved), flash_attn_func(q, k, v)), (sparse_attn_func(*moved, index), sparse_attn_func(q, k, v, index))):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
