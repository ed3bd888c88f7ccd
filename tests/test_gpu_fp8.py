"""The 8-bit layers on the GPU against 64 bits (oracle.fp8): the rounding bit for bit,
the norms and products within the bounds of their arithmetic."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import fused_linear_fp8, quantize_fp8, quantize_fp8_weight
from h3_flash_amd.fusions import (
    fused_residual_gate_rmsnorm_modulate,
    fused_residual_gate_rmsnorm_modulate_fp8,
    fused_rmsnorm_modulate,
    fused_rmsnorm_modulate_fp8,
)
from oracle.block import H, U
from oracle.fp8 import check_groups, dequantized, linear_fp8_reference, quantize_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32, E4M3, E8M0 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _randn(*shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _activations(rows, cols, seed, dtype=BF16):
    return (_randn(rows, cols, seed=seed, dtype=F32) * _randn(cols, seed=seed + 1, dtype=F32).exp()).to(dtype)


def _same(q, scale, x, block_rows=1, parts=1):
    """The pair is the reference's, NaN where it is."""
    want, byte = quantize_reference(x.reshape(-1, x.shape[-1]), block_rows, parts)
    assert q.dtype == E4M3 and scale.dtype == E8M0 and q.shape == x.shape and q.is_contiguous()
    got = scale.reshape(-1, scale.shape[-1]).view(torch.uint8).long()
    assert torch.equal(got, byte)
    assert torch.equal(q.double().reshape(want.shape).nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))


# ---------------------------------------------------------------- rounding


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, cols", [(1, 16), (1, 1024), (3, 144), (7, 5376), (129, 2064), (1000, 112), (513, 14336), (1297, 8192)])
def test_rows(rows, cols, dtype):
    x = _activations(rows, cols, rows + cols, dtype)
    _same(*quantize_fp8(x), x)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, cols, gated", [(1, 16, False), (2, 16, True), (128, 128, False), (129, 272, False), (300, 1552, True),
                                               (1000, 5376, False), (512, 256, True)])
def test_weights(rows, cols, gated, dtype):
    w = _activations(rows, cols, rows + cols, dtype)
    _same(*quantize_fp8_weight(w, gated=gated), w, 128, 2 if gated else 1)


def test_every_magnitude():
    # every bf16 value, each in a group of its own with values up to it, and
    # groups whose largest value lies next to 448 times a power of two
    bits = torch.arange(-(2**15), 2**15, dtype=torch.int32).to(torch.int16)
    top = bits.view(BF16).to(DEV)[:, None]
    x = torch.cat((top.expand(-1, 16), top.float().nan_to_num(0, 0, 0) * torch.linspace(-1, 1, 112, device=DEV)), 1).to(BF16)
    x[:, 1:16] = torch.where(torch.isfinite(x[:, 1:16]), x[:, 1:16], 0.0)
    _same(*quantize_fp8(x), x)
    edge = 448.0 * torch.exp2(torch.arange(-120, 110, device=DEV, dtype=F32))
    edge = torch.cat((edge, torch.nextafter(edge, edge * 2), torch.nextafter(edge, edge / 2)))[:, None]
    x = edge * torch.cat((torch.ones(16, device=DEV), torch.rand(112, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))))
    _same(*quantize_fp8(x), x)
    # ties: halves between neighbours of e4m3 under a scale of one
    e4m3 = torch.arange(0x7F, dtype=torch.uint8).view(E4M3).float()
    ties = torch.cat(((e4m3[1:] + e4m3[:-1]) / 2, e4m3, torch.zeros(83))).to(DEV)
    x = torch.cat((ties.view(3, 112), torch.full((3, 16), 448.0, device=DEV)), 1)
    _same(*quantize_fp8(x), x)
    _same(*quantize_fp8(-x), -x)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_that_are_not_finite(dtype):
    x = _activations(6, 400, 5, dtype)
    x[1, 3], x[2, 399], x[3, 130], x[4] = float("inf"), float("nan"), -float("inf"), 0.0
    q, s = quantize_fp8(x)
    _same(q, s, x)
    assert torch.isnan(s[1, 0].float()) and not torch.isnan(s[1, 1:].float()).any() and torch.isnan(q[1, :128].float()).all()
    assert (q[4].float() == 0).all() and (s[4].view(torch.uint8) == 1).all()
    w = _activations(260, 272, 6, dtype)
    w[200, 150] = float("nan")
    _same(*quantize_fp8_weight(w), w, 128)


def test_shapes_strides_and_offsets():
    x = _activations(24, 1040, 9)
    for view in (x.view(2, 3, 4, 1040), x[:, :512], x[::3], x.view(4, 6, 1040).transpose(0, 1), x.flatten()[3 : 3 + 24 * 1024].view(24, 1024),
                 x.t().contiguous().t(), x[0], x[:0], x[5:6, 16:48]):
        q, s = quantize_fp8(view)
        assert s.shape == (*view.shape[:-1], -(-view.shape[-1] // 128))
        if view.numel():
            _same(q, s, view.contiguous())
    _same(*quantize_fp8_weight(x[:, 16:528]), x[:, 16:528].contiguous(), 128)
    # heads of an attention output side by side
    o = _activations(10, 5 * 128, 3).view(1, 10, 5, 128)
    q, s = quantize_fp8(o.flatten(2))
    _same(q, s, o.flatten(2))


def test_a_view_of_scales_leaves_what_lies_behind_them():
    # 42 scales of a row that has room for 48
    q, s = quantize_fp8(_activations(9, 5376, 2))
    assert s.stride() == (48, 1)
    assert quantize_fp8(_activations(9, 2048, 2))[1].stride() == (16, 1)


# ---------------------------------------------------------------- norms


NORMS = [(1, 16), (3, 144), (5, 1024), (257, 5376), (64, 2064), (33, 6144), (9, 14336), (4, 16384), (130, 1008),
         # a wave per row
         (513, 5376), (515, 16), (520, 144), (600, 2064), (1001, 1008), (514, 5632)]


@pytest.mark.parametrize("tables", [BF16, F32])
@pytest.mark.parametrize("weights", [BF16, F32])
@pytest.mark.parametrize("rows, cols", NORMS)
def test_norms(rows, cols, weights, tables):
    x, r = _activations(rows, cols, rows), _randn(rows, cols, seed=2, scale=2.0)
    w = 1 + _randn(cols, seed=3, scale=0.1, dtype=weights)
    shift, scale, gate = _randn(9, 3 * cols, seed=4, scale=0.3, dtype=tables).chunk(3, -1)
    index = torch.arange(rows, device=DEV) * 9 // rows
    eps = 1e-5
    for h, got in ((x.double(), fused_rmsnorm_modulate_fp8(x, w, scale, shift, index, eps)),
                   (r.double() + gate.double()[index] * x.double(), fused_residual_gate_rmsnorm_modulate_fp8(r, x, gate, w, scale, shift, index, eps))):
        off = 4 * U * h.abs() if len(got) == 3 else 0.0 * h  # of h in fp32
        if len(got) == 3:
            off = 4 * U * (r.double().abs() + (gate.double()[index] * x.double()).abs())
            assert ((got[0].double() - h).abs() <= off + H * (h.abs() + off)).all()
        n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
        # the sum of squares to cols U of itself, its root to half that, products to a few U
        rel = (cols / 2 + 16) * U + (off.square().sum(-1, keepdim=True) / h.square().sum(-1, keepdim=True).clamp_min(1e-30)).sqrt()
        a = n * w.double() * (1 + scale.double()[index])
        y = a + shift.double()[index]
        away = a.abs() * rel + (off / h.abs().clamp_min(1e-30) * a.abs()).nan_to_num(0) + 4 * U * (a.abs() + shift.double()[index].abs())
        check_groups(got[-2], got[-1], y, away)


def test_norm_operands_anywhere():
    rows, cols = 12, 1040
    x = _activations(rows, cols + 8, 3)[:, 3 : 3 + cols]
    w = torch.cat((torch.ones(1, device=DEV), 1 + _randn(cols, seed=5, dtype=F32)))[1:]
    scale, shift, gate = (_randn(3, cols, seed=s, scale=0.3) for s in (6, 7, 8))
    index = torch.tensor([2, -1, 7, 0], dtype=torch.int32, device=DEV)
    want = fused_rmsnorm_modulate_fp8(x.contiguous(), w.clone(), scale, shift, index.long(), 1e-6)
    got = fused_rmsnorm_modulate_fp8(x, w, scale, shift, index, 1e-6)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # the bf16 forms round the same fp32 rows, but for the order of the sum of squares:
    # cols U of it at most either way, half that of its root
    near = H + cols * U
    h, n = fused_residual_gate_rmsnorm_modulate(x, x * 2, gate, w, scale, shift, index, 1e-6)
    h8, q, s = fused_residual_gate_rmsnorm_modulate_fp8(x, x * 2, gate, w, scale, shift, index, 1e-6)
    assert torch.equal(h, h8)
    check_groups(q, s, n.double(), near * n.double().abs() + 1e-30)
    n = fused_rmsnorm_modulate(x, w, scale, shift, index, 1e-6)
    check_groups(*got, n.double(), near * n.double().abs() + 1e-30)
    shaped = fused_rmsnorm_modulate_fp8(x.reshape(3, 4, cols), w, scale, shift, index, 1e-6)
    assert shaped[0].shape == (3, 4, cols) and shaped[1].shape == (3, 4, 9)
    assert torch.equal(shaped[0].reshape(rows, cols).view(torch.uint8), got[0].view(torch.uint8))
    empty = fused_rmsnorm_modulate_fp8(x[:0], w, scale, shift, index, 1e-6)
    assert empty[0].shape == (0, cols) and empty[1].shape == (0, 9)


def test_norm_of_a_row_that_is_not_finite():
    x = _activations(5, 256, 3)
    x[2, 7] = float("nan")
    ones, zeros, index = torch.ones(1, 256, device=DEV), torch.zeros(1, 256, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    q, s = fused_rmsnorm_modulate_fp8(x, ones[0], zeros, zeros, index, 1e-5)
    assert torch.isnan(s[2].float()).all() and torch.isnan(q[2].float()).all()
    assert not torch.isnan(s[[0, 1, 3, 4]].float()).any()


# ---------------------------------------------------------------- products


CASES = [
    # m, k, n, x, activation, gated, bias, residual, gate, out
    (1, 16, 8, "bf16", None, False, None, False, None, "bf16"),
    (1, 1024, 1024, "bf16", "silu", False, BF16, False, None, "bf16"),
    (1, 1024, 1024, "fp8", "silu", False, BF16, False, None, "fp8"),
    (3, 144, 40, "fp8", "gelu", False, F32, True, F32, "bf16"),
    (9, 5376, 520, "bf16", None, False, BF16, False, None, "bf16"),
    (16, 272, 264, "fp8", "silu", True, BF16, False, None, "bf16"),
    (17, 272, 272, "bf16", "gelu_tanh", True, F32, True, BF16, "fp8"),
    (31, 2064, 24, "fp8", "relu", False, None, True, None, "bf16"),
    (33, 64, 136, "bf16", "gelu", True, None, False, None, "bf16"),
    (64, 1552, 2056, "fp8", None, False, BF16, True, BF16, "bf16"),
    (65, 112, 16, "fp8", "silu", False, F32, False, None, "fp8"),
    (127, 400, 1368, "bf16", "relu", True, BF16, True, F32, "bf16"),
    (257, 1360, 272, "fp8", "gelu_tanh", False, F32, True, None, "fp8"),
    (640, 1024, 4104, "fp8", "gelu", False, BF16, False, None, "bf16"),
    (1297, 1552, 2056, "fp8", "gelu_tanh", False, F32, True, F32, "bf16"),
    (1560, 5120, 1296, "bf16", "silu", True, BF16, True, BF16, "fp8"),
    (2500, 2048, 4096, "fp8", None, False, None, True, BF16, "bf16"),
    # few tokens over wide weights
    (5, 144, 4104, "fp8", "relu", False, BF16, True, None, "bf16"),
    (20, 400, 4112, "bf16", "gelu", False, F32, True, BF16, "fp8"),
    (16, 144, 16408, "bf16", None, False, BF16, True, F32, "bf16"),
    (32, 272, 16392, "fp8", "silu", False, None, False, None, "bf16"),
    (3, 272, 8208, "fp8", "silu", True, F32, True, BF16, "fp8"),
    (27, 272, 8200, "bf16", "gelu_tanh", True, BF16, False, None, "bf16"),
    # tiles of every shape, plain and gated, with either result
    (200, 272, 8200, "fp8", "relu", False, BF16, True, None, "bf16"),
    (300, 272, 8208, "bf16", None, False, F32, True, BF16, "fp8"),
    (450, 272, 8200, "fp8", "silu", False, None, True, None, "bf16"),
    (800, 272, 14352, "fp8", "gelu", False, BF16, True, F32, "fp8"),
    (70, 272, 8200, "fp8", "gelu", True, BF16, True, None, "bf16"),
    (100, 272, 8208, "bf16", "silu", True, None, True, F32, "fp8"),
    (150, 272, 8200, "fp8", "relu", True, F32, False, None, "bf16"),
    (600, 272, 8208, "fp8", "silu", True, BF16, True, BF16, "fp8"),
    (1100, 272, 14344, "fp8", None, True, None, False, None, "bf16"),
    # long reductions: tiles in pieces, alone and after rounds of whole ones
    (40, 4112, 264, "fp8", "gelu_tanh", False, BF16, True, BF16, "bf16"),
    (40, 4112, 272, "bf16", "silu", True, F32, True, F32, "fp8"),
    (70, 8208, 2696, "fp8", None, False, BF16, False, None, "bf16"),
    (70, 8208, 1040, "fp8", "gelu", True, None, True, None, "fp8"),
    (200, 8208, 1032, "bf16", "silu", True, BF16, False, None, "bf16"),
    (450, 8208, 8200, "fp8", None, False, BF16, True, F32, "bf16"),
    (390, 5376, 5376, "bf16", None, False, None, True, F32, "bf16"),
    (3120, 14352, 5368, "fp8", None, False, F32, True, BF16, "bf16"),
    (3120, 4112, 8208, "fp8", "silu", True, None, False, None, "fp8"),
    (1560, 14336, 5376, "fp8", None, False, BF16, True, BF16, "bf16"),
]


def _operands(m, k, n, x, gated, seed=0):
    rows = 2 * n if gated else n
    a = _activations(m, k, seed + m)
    w = quantize_fp8_weight(_randn(rows, k, seed=seed + k, scale=k**-0.5), gated=gated)
    return (a, None, *w) if x == "bf16" else (*quantize_fp8(a), *w)


def _check(got, quantize, x, x_scale, w, w_scale, bias, **kwargs):
    want, bound = linear_fp8_reference(x, w, w_scale, bias, x_scale=x_scale, rounded=not quantize, **kwargs)
    if quantize:
        q, s = (t.reshape(-1, t.shape[-1]) for t in got)
        check_groups(q, s, want, bound)
        rel = (dequantized(q, s) - want).norm() / want.norm()
        assert rel < 0.04, rel  # half a step of e4m3: 2^-4 at most, 2^-4 / sqrt(6) over all mantissas
        return
    assert got.dtype == BF16
    off = (got.double().reshape(want.shape) - want).abs()
    worst = (off / bound).nan_to_num(nan=float("inf")).max().item()
    assert worst <= 1.0, worst
    # over all mantissas a rounding to bf16 is off by 2^-8 / sqrt(6)
    rel = (off.norm() / want.norm()).item() if want.numel() > 4096 else 0.0
    assert rel < 0.0022, rel


@pytest.mark.parametrize("m, k, n, x, activation, gated, bias, residual, gate, out", CASES)
def test_products(m, k, n, x, activation, gated, bias, residual, gate, out):
    a, a_scale, w, w_scale = _operands(m, k, n, x, gated)
    rows = 2 * n if gated else n
    b = None if bias is None else _randn(rows, seed=1, scale=0.3, dtype=bias)
    r = _randn(m, n, seed=2, scale=2.0) if residual else None
    g = None if gate is None else _randn(9, n, seed=3, dtype=gate)
    index = None if gate is None else torch.arange(m, device=DEV) * 9 // m
    rest = dict(activation=activation, gated=gated, residual=r, gate=g, index=index)
    got = fused_linear_fp8(a, w, w_scale, b, x_scale=a_scale, quantize=out == "fp8", **rest)
    _check(got, out == "fp8", a, a_scale, w, w_scale, b, **rest)
    again = fused_linear_fp8(a, w, w_scale, b, x_scale=a_scale, quantize=out == "fp8", **rest)
    for one, two in zip(*((t if out == "fp8" else (t,)) for t in (got, again))):
        assert torch.equal(one.view(torch.uint8), two.view(torch.uint8))


@pytest.mark.parametrize("m", [1, 16, 17, 32, 33, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_bf16_rows_are_rounded_as_quantize_fp8_does(m, gated):
    a, _, w, w_scale = _operands(m, 1360, 272, "bf16", gated)
    got = fused_linear_fp8(a, w, w_scale, gated=gated, activation="silu")
    q, s = quantize_fp8(a)
    assert torch.equal(got, fused_linear_fp8(q, w, w_scale, x_scale=s, gated=gated, activation="silu"))


@pytest.mark.parametrize("m", [1, 20, 40, 200])
def test_extreme_scales(m):
    # operands at both ends of their range, whose product lies within bf16's
    k, n = 272, 144
    a, w = _activations(m, k, 3, F32), _randn(n, k, seed=4, dtype=F32)
    a, w = a * 2.0**-110, w * 2.0**100
    a[:, 128:256] *= 2.0**60
    w[:, 128:256] *= 2.0**-60
    (q, s), (wq, ws) = quantize_fp8(a), quantize_fp8_weight(w)
    _check(fused_linear_fp8(q, wq, ws, x_scale=s), False, q, s, wq, ws, None)


@pytest.mark.parametrize("m", [2, 20, 40, 300])
@pytest.mark.parametrize("x", ["bf16", "fp8"])
def test_values_that_are_not_finite_stay_in_their_row(m, x):
    k, n = 400, 272
    a = _activations(m, k, 3)
    a[1, 170] = float("nan")
    w, ws = quantize_fp8_weight(_randn(n, k, seed=4, scale=0.05))
    q, s = quantize_fp8(a) if x == "fp8" else (a, None)
    y = fused_linear_fp8(q, w, ws, x_scale=s)
    assert torch.isnan(y[1]).all() and not torch.isnan(y[[0, *range(2, m)]]).any()
    yq, ys = fused_linear_fp8(q, w, ws, x_scale=s, quantize=True)
    assert torch.isnan(ys[1].float()).all() and torch.isnan(yq[1].float()).all() and not torch.isnan(ys[0].float()).any()


@pytest.mark.parametrize("m", [5, 70, 300])
def test_operands_anywhere(m):
    k, n = 400, 272
    a, a_scale, w, w_scale = _operands(m, k, n, "fp8", False)
    want = fused_linear_fp8(a, w, w_scale, x_scale=a_scale)
    wide = torch.zeros((m, 432), dtype=torch.uint8, device=DEV)
    wide[:, 7 : 7 + k] = a.view(torch.uint8)
    ws = torch.zeros((w_scale.shape[0], 7), dtype=torch.uint8, device=DEV)
    ws[:, 2 : 2 + w_scale.shape[1]] = w_scale.view(torch.uint8)
    xs = torch.zeros((a_scale.shape[1], m), dtype=torch.uint8, device=DEV)
    xs[:] = a_scale.view(torch.uint8).t()
    got = fused_linear_fp8(wide[:, 7 : 7 + k].view(E4M3), w, ws[:, 2:6].view(E8M0), x_scale=xs.t().view(E8M0))
    assert torch.equal(got, want)
    got = fused_linear_fp8(a, w.t().contiguous().t(), w_scale.contiguous(), x_scale=a_scale.contiguous())
    assert torch.equal(got, want)
    # into rows of a wider result, the columns beside them left as they were
    out = torch.full((m, n + 64), 7.0, dtype=BF16, device=DEV)
    assert fused_linear_fp8(a, w, w_scale, x_scale=a_scale, out=out[:, 32 : 32 + n]).data_ptr() == out[:, 32:].data_ptr()
    assert torch.equal(out[:, 32 : 32 + n], want) and (out[:, :32] == 7).all() and (out[:, 32 + n :] == 7).all()
    # onto the residual itself
    r = _randn(m, n, seed=8)
    want = fused_linear_fp8(a, w, w_scale, x_scale=a_scale, residual=r)
    fused_linear_fp8(a, w, w_scale, x_scale=a_scale, residual=r, out=r)
    assert torch.equal(r, want)


def test_leading_dimensions_and_no_rows():
    a, a_scale, w, w_scale = _operands(24, 272, 144, "fp8", False)
    want = fused_linear_fp8(a, w, w_scale, x_scale=a_scale)
    got = fused_linear_fp8(a.view(2, 3, 4, 272), w, w_scale, x_scale=a_scale.view(2, 3, 4, 3))
    assert got.shape == (2, 3, 4, 144) and torch.equal(got.view(24, 144), want)
    q, s = fused_linear_fp8(a.view(2, 3, 4, 272), w, w_scale, x_scale=a_scale.view(2, 3, 4, 3), quantize=True)
    assert q.shape == (2, 3, 4, 144) and s.shape == (2, 3, 4, 2)
    one = fused_linear_fp8(a[3], w, w_scale, x_scale=a_scale[3])
    assert one.shape == (144,) and torch.equal(one, fused_linear_fp8(a[3:4], w, w_scale, x_scale=a_scale[3:4])[0])
    assert fused_linear_fp8(a[:0], w, w_scale, x_scale=a_scale[:0]).shape == (0, 144)
    q, s = fused_linear_fp8(a[:0], w, w_scale, x_scale=a_scale[:0], quantize=True)
    assert q.shape == (0, 144) and s.shape == (0, 2)


@pytest.mark.parametrize("m", [4, 300])
def test_index_and_other_streams(m):
    a, a_scale, w, w_scale = _operands(m, 400, 272, "fp8", False)
    g, r = _randn(5, 272, seed=3, dtype=F32), _randn(m, 272, seed=4)
    index = torch.tensor([4, -3, 9, 1, 0, 2, 2], dtype=torch.int32, device=DEV)
    got = fused_linear_fp8(a, w, w_scale, x_scale=a_scale, residual=r, gate=g, index=index)
    _check(got, False, a, a_scale, w, w_scale, None, residual=r, gate=g, index=index)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = fused_linear_fp8(a, w, w_scale, x_scale=a_scale, residual=r, gate=g, index=index.long())
        q, s = quantize_fp8(there)
    side.synchronize()
    assert torch.equal(there, got)
    _same(q, s, got)
