"""Forms of the 8-bit product that the other files' sizes do not take, against 64 bits:
reductions longer than the scales that a tile holds at once (a ring whose slots are loaded
again, registers that are filled again), in every tile shape and split, and the few-token
form in every block count and pair of types. tests/test_fp8_forms_host.py asks the plan
which form each takes."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import fused_linear_fp8
from test_gpu_fp8 import BF16, DEV, F32, _check, _operands, _randn

pytestmark = pytest.mark.gpu

# m, k, n, gated, 8-bit result: the scales in turn, but where noted
CASES = [
    # 128 features x 32, 64, 96 and 128 tokens, whole
    (20, 16304, 8808, True, False), (285, 17456, 5520, False, False), (67, 14768, 11072, True, False), (5485, 14960, 296, False, False),
    (99, 15168, 11776, True, False), (201, 15376, 11376, False, False),
    # pieces behind rounds of whole tiles
    (259, 15200, 6152, True, False), (262, 17984, 10992, False, False), (423, 15456, 5432, True, False), (4721, 14928, 872, False, False),
    # 256 features x 128, 192 and 256 tokens, whole
    (387, 16080, 5560, True, False), (417, 15392, 11080, False, False), (263, 10688, 22128, False, True), (1566, 6272, 7200, False, False),
    # pieces
    (129, 22016, 11976, True, False), (346, 20752, 11656, False, False), (434, 19040, 4384, True, False), (780, 19488, 4776, False, False),
    # pieces behind rounds of whole tiles (the first: the scales at once)
    (982, 11888, 8216, False, False), (403, 15456, 8560, True, False), (5439, 14624, 1440, False, False), (659, 10848, 8288, True, False),
    (5378, 10384, 2112, False, False), (1179, 6224, 7152, True, False),
]

# m, k, n, gated, x, 8-bit result
FEW_TOKENS = [
    # one, two and four blocks of 16 features x 16 tokens
    (7, 1552, 272, False, "bf16", True), (5, 1040, 16, True, "fp8", True), (16, 2064, 144, True, "bf16", True), (1, 1360, 40, True, "bf16", False),
    (3, 400, 5728, False, "fp8", True), (9, 272, 4176, False, "bf16", True), (15, 1040, 4120, False, "bf16", False),
    (2, 208, 8272, True, "bf16", True), (11, 272, 10600, True, "fp8", False), (6, 400, 9272, True, "bf16", False),
    (13, 208, 21248, False, "fp8", True), (4, 224, 18032, False, "bf16", True),
    # x 32 tokens
    (18, 1552, 144, False, "fp8", True), (31, 1040, 272, False, "bf16", True), (17, 2064, 264, False, "bf16", False),
    (29, 1360, 16, True, "fp8", True), (32, 400, 136, True, "fp8", False), (19, 1040, 24, True, "bf16", False),
    (21, 272, 4176, False, "fp8", True), (30, 208, 4776, False, "fp8", False), (25, 400, 4336, False, "bf16", False),
    (18, 208, 8384, True, "fp8", True), (27, 224, 8608, True, "bf16", True), (23, 208, 8952, True, "fp8", False),
    (26, 208, 17184, False, "fp8", True), (20, 224, 16928, False, "bf16", True),
]


def _product(i, m, k, n, gated, x, quantize):
    a, a_scale, w, w_scale = _operands(m, k, n, x, gated)
    rows = 2 * n if gated else n
    # the epilogue's parts in turn: none, a bias, all of them, a residual
    b = _randn(rows, seed=1, scale=0.3, dtype=(BF16, F32)[i % 2]) if i % 4 in (1, 2) else None
    r = _randn(m, n, seed=2, scale=2.0) if i % 4 > 1 else None
    g = _randn(7, n, seed=3, dtype=(F32, BF16)[i % 2]) if i % 4 == 2 else None
    index = None if g is None else torch.arange(m, device=DEV, dtype=(torch.int32, torch.int64)[i % 2]) * 7 // m
    rest = dict(activation=(None, "silu", "gelu", "gelu_tanh", "relu")[i % 5], gated=gated, residual=r, gate=g, index=index)
    got = fused_linear_fp8(a, w, w_scale, b, x_scale=a_scale, quantize=quantize, **rest)
    _check(got, quantize, a, a_scale, w, w_scale, b, **rest)
    again = fused_linear_fp8(a, w, w_scale, b, x_scale=a_scale, quantize=quantize, **rest)
    for one, two in zip(*((t if quantize else (t,)) for t in (got, again))):
        assert torch.equal(one.view(torch.uint8), two.view(torch.uint8))


@pytest.mark.parametrize("m, k, n, gated, quantize", CASES)
def test_tiles(m, k, n, gated, quantize):
    _product(CASES.index((m, k, n, gated, quantize)), m, k, n, gated, "fp8", quantize)


@pytest.mark.parametrize("m, k, n, gated, x, quantize", FEW_TOKENS)
def test_few_tokens(m, k, n, gated, x, quantize):
    _product(FEW_TOKENS.index((m, k, n, gated, x, quantize)), m, k, n, gated, x, quantize)
