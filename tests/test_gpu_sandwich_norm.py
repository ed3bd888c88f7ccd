"""GPU parity of the norms before and after a branch against 64 bits, elementwise
within the bound of fp32 arithmetic and one rounding (oracle.block)."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd.fusions import (
    fused_residual_gate_rmsnorm_modulate,
    fused_rmsnorm_residual_gate_rmsnorm_modulate,
)
from oracle.block import sandwich_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32 = torch.bfloat16, torch.float32


def _inputs(rows, cols, tables=BF16, weights=BF16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(1000 * rows + cols + seed)
    randn = lambda *s: torch.randn(s, device=DEV, generator=g)  # noqa: E731
    wide = (0.3 * randn(9, 3 * cols)).to(tables).chunk(3, -1)
    return {
        "residual": (2 * randn(rows, cols)).to(BF16),
        "branch": randn(rows, cols).to(BF16),
        "branch_weight": (1 + 0.1 * randn(cols)).to(weights),
        "gate": wide[0],
        "weight": (1 + 0.1 * randn(cols)).to(weights),
        "scale": wide[1],
        "shift": wide[2],
        "index": torch.arange(rows, device=DEV) % 9,
    }


def _check(got, want):
    for name, y, (ref, bound) in zip(("hidden", "normed"), got, (want[:2], want[2:])):
        if ref is None:
            assert y is None
            continue
        assert y.dtype == BF16
        worst = ((y.double().reshape(ref.shape) - ref).abs() / bound).nan_to_num(nan=float("inf")).max().item()
        assert worst <= 1.0, (name, worst)


def _run(a, eps=1e-5, **kwargs):
    return fused_rmsnorm_residual_gate_rmsnorm_modulate(*a.values(), eps, **kwargs)


@pytest.mark.parametrize(
    "rows, cols, tables, weights, scale",
    [
        (1, 8, BF16, BF16, 1.0),
        (257, 5376, BF16, BF16, 1.0),
        (33, 1000, F32, F32, 0.5),
        (17, 1001, BF16, F32, 1.0),  # odd width: element form
        (5, 20000, BF16, BF16, -1.25),  # wider than the vector forms
        (6, 512, BF16, F32, 0.0),
        (7, 520, BF16, BF16, 1.0),  # a second vector on one lane
        (10, 5632, BF16, F32, 2.0),
        (7, 5640, BF16, BF16, 1.0),
        (9, 2056, F32, BF16, 1.0),
        (3, 8192, F32, F32, 1.0),
        (4, 8200, F32, BF16, 1.0),
        (1297, 1024, BF16, BF16, 1.0),
        (3, 16384, BF16, F32, 1.0),
        (2, 12296, F32, BF16, 1.0),
        # one wave per row (past 1,024 rows, up to 4,096 columns), its last rows
        # and vectors partial
        (1025, 8, BF16, BF16, 1.0),
        (1026, 1000, BF16, F32, 0.5),
        (1027, 2056, BF16, BF16, 1.0),
        (1029, 3600, BF16, F32, 1.0),
        (1030, 4096, BF16, BF16, 1.0),
        # two waves per row (past 16,384 rows)
        (16385, 4104, BF16, BF16, 1.0),
        (16387, 5376, BF16, F32, 0.75),
        (16386, 7168, BF16, BF16, 1.0),
    ],
)
def test_parity(rows, cols, tables, weights, scale):
    a = _inputs(rows, cols, tables, weights)
    got = _run(a, residual_scale=scale)
    assert got[0].shape == got[1].shape == (rows, cols)
    _check(got, sandwich_reference(*a.values(), 1e-5, scale))


@pytest.mark.parametrize("rows, cols", [(19, 24), (19, 1001), (19, 5376), (1031, 640), (16389, 4200)])
def test_without_gate_or_second_norm(rows, cols):
    a = _inputs(rows, cols)
    a["gate"] = None
    _check(_run(a), sandwich_reference(*a.values(), 1e-5))
    a = _inputs(rows, cols)
    a["weight"] = a["scale"] = a["shift"] = None
    _check(_run(a), sandwich_reference(*a.values(), 1e-5))
    a["gate"] = a["index"] = None
    hidden, normed = _run(a, residual_scale=0.5)
    assert normed is None
    _check((hidden, None), sandwich_reference(*a.values(), 1e-5, 0.5))


@pytest.mark.parametrize("cols", [2048, 1001])
def test_strides_broadcast_rows_and_index_outside_the_table(cols):
    a = _inputs(40, cols)
    wide = torch.randn((40, cols + 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(7)).to(BF16)
    a["branch"] = wide[:, :cols]
    a["gate"] = a["gate"][:1].expand(9, cols)
    a["index"] = torch.tensor([0, 3, 8, 12, -1], dtype=torch.int32, device=DEV)
    _check(_run(a), sandwich_reference(*a.values(), 1e-5))


def test_mixed_dtypes_and_batches():
    a = _inputs(24, 512)
    a["branch_weight"], a["scale"] = a["branch_weight"].float(), a["scale"].float()
    for name in ("residual", "branch"):
        a[name] = a[name].view(2, 12, 512)
    got = _run(a)
    assert got[0].shape == got[1].shape == (2, 12, 512)
    _check(got, sandwich_reference(*a.values(), 1e-5))


@pytest.mark.parametrize("cols", [5120, 1001])
def test_edge_magnitudes(cols):
    # a branch of zeros, tiny and large values, squares that overflow fp32 (its
    # norm factor goes to 0), and a row that is zero altogether
    a = _inputs(6, cols)
    a["branch"][0] = 0.0
    a["branch"][1] *= 1e-30
    a["branch"][2] *= 1e17
    a["branch"][3] = 0.0
    a["residual"][3] = 0.0
    got = _run(a, eps=1e-6)
    _check(got, sandwich_reference(*a.values(), 1e-6))
    a["branch"][4] *= 1e30
    hidden, _ = _run(a, eps=1e-6)
    assert torch.equal(hidden[4], a["residual"][4])
    # a row that is not finite stays alone
    a["branch"][5, 3] = float("nan")
    again, _ = _run(a, eps=1e-6)
    assert torch.equal(again[:5], hidden[:5]) and again[5].isnan().all()


def test_unit_branch_norm_matches_the_variant_without_it():
    # rows of +-1 are their own norm (eps 0): the same as without the first norm
    a = _inputs(12, 1024)
    a["branch"] = torch.where(a["branch"] > 0, 1.0, -1.0).to(BF16)
    a["branch_weight"] = torch.ones(1024, dtype=BF16, device=DEV)
    hidden, normed = _run(a, eps=0.0)
    want = fused_residual_gate_rmsnorm_modulate(
        a["residual"], a["branch"], a["gate"], a["weight"], a["scale"], a["shift"], a["index"], 0.0
    )
    assert torch.equal(hidden, want[0])
    # (another order of the second sum: a step of bf16 at a rounding border)
    assert ((normed.float() - want[1].float()).abs() <= 2.0**-7 * want[1].float().abs() + 1e-6).all()


def test_empty_and_refusals():
    a = _inputs(4, 64)
    empty = dict(a, residual=a["residual"][:0], branch=a["branch"][:0])
    assert _run(empty)[1].shape == (0, 64)
    for change, kind in (
        ({"residual": a["residual"].float()}, TypeError),
        ({"branch": a["branch"][:3]}, ValueError),
        ({"branch_weight": a["branch_weight"][:32]}, ValueError),
        ({"weight": None}, ValueError),
        ({"shift": None}, ValueError),
        ({"gate": a["gate"][:, :32]}, ValueError),
        ({"index": None}, ValueError),
        ({"index": a["index"][:0]}, ValueError),
    ):
        with pytest.raises(kind):
            _run(dict(a, **change))
    with pytest.raises(ValueError):
        _run(a, eps=-1.0)
    with pytest.raises(ValueError):
        _run(a, residual_scale=float("inf"))
