"""GPU parity of the linear layer with its epilogue against 64 bits, elementwise
within the bound of fp32 accumulation and one rounding (oracle.block)."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import fused_linear
from h3_flash_amd.fusions import fused_swiglu
from oracle.block import linear_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32 = torch.bfloat16, torch.float32


def _randn(*shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _check(got, x, weight, *args, tag="", **kwargs):
    want, bound = linear_reference(x, weight, *args, **kwargs)
    assert got.dtype == BF16
    off = (got.double().reshape(want.shape) - want).abs()
    worst = (off / bound).nan_to_num(nan=float("inf")).max().item()
    assert worst <= 1.0, (tag, worst)


CASES = [
    # m, k, n, activation, gated, bias, residual, gate
    (1, 8, 8, None, False, None, False, None),
    (1, 1024, 1024, "silu", False, BF16, False, None),
    (3, 72, 40, "gelu", False, F32, True, F32),
    (9, 5376, 520, None, False, BF16, False, None),
    (16, 136, 264, "silu", True, BF16, False, None),
    (17, 136, 264, "gelu_tanh", True, F32, True, BF16),
    (31, 2056, 24, "relu", False, None, True, None),
    (33, 64, 136, "gelu", True, None, False, None),
    (64, 1544, 2056, None, False, BF16, True, BF16),
    (65, 56, 8, "silu", False, F32, False, None),
    (127, 200, 1368, "relu", True, BF16, True, F32),
    (257, 1352, 264, "gelu_tanh", False, F32, True, None),
    (640, 1024, 4104, "gelu", False, BF16, False, None),
    (1297, 1544, 2056, "gelu_tanh", False, F32, True, F32),
    (1560, 5120, 1288, "silu", True, BF16, True, BF16),
    (2500, 2048, 4096, None, False, None, True, BF16),
    # few tokens over wide weights: two and four blocks of rows per workgroup
    (5, 72, 4104, "relu", False, BF16, True, None),
    (20, 200, 4104, "gelu", False, F32, True, BF16),
    (16, 72, 16408, None, False, BF16, True, F32),
    (32, 264, 16392, "silu", False, None, False, None),
    (3, 136, 8200, "silu", True, F32, True, BF16),
    (27, 136, 8200, "gelu_tanh", True, BF16, False, None),
    # every tile shape, plain and gated
    (200, 264, 8200, "relu", False, BF16, True, None),
    (300, 264, 8200, None, False, F32, True, BF16),
    (450, 264, 8200, "silu", False, None, True, None),
    (800, 264, 14344, "gelu", False, BF16, True, F32),
    (70, 264, 8200, "gelu", True, BF16, True, None),
    (100, 264, 8200, "silu", True, None, True, F32),
    (150, 264, 8200, "relu", True, F32, False, None),
    (600, 264, 8200, "silu", True, BF16, True, BF16),
    (1100, 264, 14344, None, True, None, False, None),
    # tiles in pieces along k: alone, and after rounds of whole tiles; k ends
    # inside the last piece's last step
    (40, 4104, 264, "gelu_tanh", False, BF16, True, BF16),
    (40, 4104, 264, "silu", True, F32, True, F32),
    (70, 8200, 2696, None, False, BF16, False, None),
    (70, 8200, 1032, "gelu", True, None, True, None),
    (100, 8200, 4104, "relu", False, F32, True, BF16),
    (200, 8200, 1032, "silu", True, BF16, False, None),
    (150, 4104, 8200, "silu", True, None, True, BF16),
    (450, 8200, 8200, None, False, BF16, True, F32),
    (450, 8200, 8200, "silu", True, None, False, None),
    (3120, 4104, 2696, "gelu", True, BF16, True, BF16),
    (3120, 14344, 5368, None, False, F32, True, BF16),
    (3120, 4104, 8200, "silu", True, None, False, None),
    (4100, 8200, 1032, "relu", False, BF16, True, None),
    (1560, 14336, 5376, None, False, BF16, True, BF16),
    (100, 264, 8200, "gelu_tanh", False, None, True, F32),
    (40, 264, 8200, None, True, BF16, True, None),
]


@pytest.mark.parametrize("m, k, n, activation, gated, bias, residual, gate", CASES)
def test_parity(m, k, n, activation, gated, bias, residual, gate):
    rows = 2 * n if gated else n
    x, w = _randn(m, k, seed=m), _randn(rows, k, seed=k, scale=k**-0.5)
    b = None if bias is None else _randn(rows, seed=1, scale=0.3, dtype=bias)
    r = _randn(m, n, seed=2, scale=2.0) if residual else None
    g = None if gate is None else _randn(9, n, seed=3, dtype=gate)
    index = None if gate is None else torch.arange(m, device=DEV) * 9 // m
    got = fused_linear(x, w, b, activation=activation, gated=gated, residual=r, gate=g, index=index)
    assert got.shape == (m, n)
    _check(got, x, w, b, activation, gated, r, g, index)


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh", "relu"])
def test_activations_over_their_range(m, activation):
    # the product is the first column of x: values from far tails to overflow
    values = torch.cat((torch.linspace(-12, 12, 4096), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 40.0, -40.0, 1e19, -1e19, 3e38, -3e38])))
    values = torch.cat((values, torch.zeros(-len(values) % 8))).to(BF16)
    x = torch.zeros((m, 8), dtype=BF16)
    x[:, 0] = 1.0
    w = torch.zeros((len(values), 8), dtype=BF16)
    w[:, 0] = values
    got = fused_linear(x.to(DEV), w.to(DEV), activation=activation)
    _check(got.cpu(), x, w, None, activation)
    inf = w.clone()
    inf[:, 0] = torch.tensor([float("inf"), -float("inf")], dtype=BF16).repeat(len(values) // 2)
    x[:, 1:] = 0.0
    inf[:, 1:] = 0.0
    ends = fused_linear(x.to(DEV), inf.to(DEV), activation=activation).cpu()[0, :2].float()
    assert ends[0] == float("inf")
    assert ends[1] == (-float("inf") if activation is None else 0.0)
    nan = w.clone()
    nan[3, 0] = float("nan")
    got = fused_linear(x.to(DEV), nan.to(DEV), activation=activation).cpu()
    assert got[:, 3].isnan().all() and not got[:, :3].isnan().any() and not got[:, 4:].isnan().any()


@pytest.mark.parametrize("m", [4, 40, 200])
def test_what_lies_beside_the_operands_is_not_read_into_them(m):
    # k ends inside a K step and a 128-byte line; the columns after it, rows past
    # the tensors and the last rows hold NaN
    k, n = 72, 24
    xs = torch.full((m + 3, k + 16), float("nan"), dtype=BF16, device=DEV)
    ws = torch.full((n + 5, k + 24), float("nan"), dtype=BF16, device=DEV)
    xs[:m, :k], ws[:n, :k] = _randn(m, k, seed=4), _randn(n, k, seed=5)
    ys = torch.full((m + 2, n + 8), 7.0, dtype=BF16, device=DEV)
    got = fused_linear(xs[:m, :k], ws[:n, :k], activation="silu", out=ys[:m, :n])
    _check(got, xs[:m, :k], ws[:n, :k], None, "silu")
    assert (ys[m:] == 7.0).all() and (ys[:, n:] == 7.0).all()


@pytest.mark.parametrize("m", [6, 130])
def test_one_token_or_feature_does_not_touch_another(m):
    k, n = 264, 144
    x, w = _randn(m, k, seed=6), _randn(n, k, seed=7)
    clean = fused_linear(x, w)
    x[2], w[5] = float("nan"), float("inf")
    got = fused_linear(x, w)
    keep = torch.ones((m, n), dtype=torch.bool, device=DEV)
    keep[2], keep[:, 5] = False, False
    assert torch.equal(got[keep], clean[keep])
    assert got[2].isnan().all() and not torch.isfinite(got[:, 5]).any()


@pytest.mark.parametrize("m", [7, 150])
def test_views_batches_and_index_forms(m):
    k, n = 128, 96
    x = _randn(2, m, 3 * k, seed=8)[:, :, k : 2 * k]  # a chunk of a wider tensor
    w = _randn(2 * n, k + 8, seed=9, scale=k**-0.5)[:, :k]
    residual = _randn(2, m, 2 * n, seed=10)[..., n:]
    gate = _randn(1, n, seed=11, dtype=F32).expand(4, n)
    index = torch.tensor([0, 7, -2, 3, 1], dtype=torch.int32, device=DEV)  # 7 and -2 outside the table
    got = fused_linear(x, w, gated=True, activation="silu", residual=residual, gate=gate, index=index)
    assert got.shape == (2, m, n)
    _check(got, x, w, None, "silu", True, residual, gate, index)
    turned = _randn(k, 2 * n, seed=12, scale=k**-0.5).t()  # columns contiguous: copied
    _check(fused_linear(x, turned, _randn(2 * n + 3, seed=13)[3:]), x, turned, _randn(2 * n + 3, seed=13)[3:])


@pytest.mark.parametrize("m", [5, 90, 300])
def test_out_may_be_the_residual(m):
    x, w, r = _randn(m, 264, seed=14), _randn(136, 264, seed=15, scale=0.06), _randn(m, 136, seed=16)
    apart = fused_linear(x, w, residual=r)
    assert fused_linear(x, w, residual=r, out=r).data_ptr() == r.data_ptr()
    assert torch.equal(r, apart)


def test_forms_agree_with_the_separate_steps():
    # the gated product against the GEMM and the swiglu kernel, which round once more
    x, w = _randn(333, 512, seed=17), _randn(2 * 640, 512, seed=18, scale=512**-0.5)
    steps = fused_swiglu(fused_linear(x, w))
    fused = fused_linear(x, w, gated=True, activation="silu")
    # rounding value and gate to bf16 first: 2 halves of a step and the slope of silu
    assert ((steps.float() - fused.float()).abs() <= 2.0**-6 * fused.float().abs() + 2.0**-7).all()


def test_empty_batch():
    w = _randn(16, 24, seed=19)
    assert fused_linear(torch.empty((0, 24), dtype=BF16, device=DEV), w).shape == (0, 16)
    assert fused_linear(torch.empty((2, 0, 24), dtype=BF16, device=DEV), w, gated=True).shape == (2, 0, 8)


def test_refusals():
    x, w = _randn(4, 64, seed=20), _randn(32, 64, seed=21)
    index = torch.zeros(1, dtype=torch.long, device=DEV)
    for kind, args, kwargs in (
        (TypeError, (x.float(), w), {}),
        (TypeError, (x, w.float()), {}),
        (ValueError, (x[:, :56], w), {}),
        (ValueError, (x[:, :60], w[:, :60]), {}),
        (ValueError, (x, w[:20]), {}),
        (ValueError, (x, w[:24]), {"gated": True}),
        (ValueError, (x, w[:31]), {"gated": True}),
        (ValueError, (x, w), {"activation": "tanh"}),
        (ValueError, (x, w, torch.zeros(31, device=DEV)), {}),
        (ValueError, (x, w), {"residual": _randn(4, 24, seed=1)}),
        (ValueError, (x, w), {"gate": _randn(2, 32, seed=1)}),
        (ValueError, (x, w), {"gate": _randn(2, 24, seed=1), "index": index}),
        (ValueError, (x, w), {"gate": _randn(2, 32, seed=1), "index": index[:0]}),
        (ValueError, (x, w), {"out": torch.empty((4, 32), device=DEV)}),
        (ValueError, (x, w), {"out": torch.empty((32, 4), dtype=BF16, device=DEV).t()}),
    ):
        with pytest.raises(kind):
            fused_linear(*args, **kwargs)
