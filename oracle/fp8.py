"""64-bit restatement of the 8-bit layers: rounding to e4m3 with a power of two for a
group, and the matrix product of such operands — test infrastructure only."""

from __future__ import annotations

import torch

from .block import U, linear_reference

__all__ = ["GROUP", "SUMS", "check_groups", "dequantized", "linear_fp8_reference", "quantize_reference", "scale_byte"]

GROUP = 128
# The matrix cores line the products of 8 neighbouring K up to the largest, whose
# leading bit they keep 13 bits below: each of the 7 others is off by at most 2^-13 of
# it, and a sum of such groups by 7 * 2^-13 of the sum of all magnitudes (their own
# width, 24 bits, is in linear_reference's bound).
SUMS = 7 * 2.0**-13


def scale_byte(top: torch.Tensor) -> torch.Tensor:
    """e of the smallest 2^(e - 127) >= top / 448, at least 1; 255 where top is not finite."""
    part, power = torch.frexp(top.double())  # part in [1/2, 1)
    e = power + 127 - 9 + (part > 0.875).to(power.dtype)  # 448 = 0.875 * 2^9
    e = torch.where(top == 0, 1, e.clamp(1, 254))
    return torch.where(torch.isfinite(top), e, 255).to(torch.int64)


def _value(byte: torch.Tensor) -> torch.Tensor:
    return torch.where(byte == 255, torch.nan, torch.exp2(byte.double() - 127))


def _rows_of_blocks(rows: int, block_rows: int, parts: int) -> torch.Tensor:
    """The scale row of each row."""
    per = rows // parts
    r = torch.arange(rows)
    return r // per * (-(-per // block_rows)) + r % per // block_rows


def _e4m3(v: torch.Tensor) -> torch.Tensor:
    step = torch.exp2(torch.frexp(v.abs().clamp_min(2.0**-6))[1].double() - 1 - 3)
    return torch.round(v / step) * step


def quantize_reference(x: torch.Tensor, block_rows: int = 1, parts: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, byte)`` of a 2-D tensor: e4m3's values in float64, e8m0's bytes."""
    x = x.double()
    rows, cols = x.shape
    of = _rows_of_blocks(rows, block_rows, parts).to(x.device)
    blocks = int(of.max()) + 1 if rows else 0
    top = torch.zeros((blocks, -(-cols // GROUP)), dtype=torch.float64, device=x.device)
    for j in range(top.shape[1]):
        size = x[:, j * GROUP : (j + 1) * GROUP].abs()
        size = torch.where(torch.isnan(size), torch.inf, size).amax(1)
        top[:, j].scatter_reduce_(0, of, size, "amax")
    byte = scale_byte(top)
    return _e4m3(x / _value(byte)[of].repeat_interleave(GROUP, 1)[:, :cols]), byte


def dequantized(q: torch.Tensor, scale: torch.Tensor, block_rows: int = 1, parts: int = 1) -> torch.Tensor:
    """The values of a 2-D pair, in float64."""
    of = _rows_of_blocks(q.shape[0], block_rows, parts).to(q.device)
    return q.double() * _value(scale.view(torch.uint8).long())[of].repeat_interleave(GROUP, 1)[:, : q.shape[1]]


def linear_fp8_reference(x, weight, weight_scale, bias=None, *, x_scale=None, gated=False, rounded=True, **kwargs):
    """``(y, bound)`` of the product of 8-bit operands; a bf16 x is rounded first."""
    if x_scale is None:
        q, byte = quantize_reference(x.reshape(-1, x.shape[-1]))
        x = q * _value(byte).repeat_interleave(GROUP, 1)[:, : q.shape[1]]
    else:
        x = dequantized(x.reshape(-1, x.shape[-1]), x_scale.reshape(-1, x_scale.shape[-1]))
    w = dequantized(weight, weight_scale, GROUP, 2 if gated else 1)
    return linear_reference(x, w, bias, gated=gated, sums=SUMS, rounded=rounded, **kwargs)


def check_groups(q: torch.Tensor, scale: torch.Tensor, y: torch.Tensor, off: torch.Tensor) -> None:
    """Asserts that a 2-D pair is the rounding of values within ``off`` of ``y``: its
    scales are those of some largest magnitude in reach, its values off by half a step
    (2^-4 of the value, 2^-10 of the scale where that is more)."""
    byte = scale.view(torch.uint8).long()
    for j in range(byte.shape[1]):
        at = slice(j * GROUP, (j + 1) * GROUP)
        lo, hi = ((y[:, at].abs() + s * off[:, at]).clamp_min(0.0).amax(1) for s in (-1, 1))
        assert (byte[:, j] >= scale_byte(lo)).all() and (byte[:, j] <= scale_byte(hi)).all(), j
    s = _value(byte).repeat_interleave(GROUP, 1)[:, : q.shape[1]]
    half = torch.maximum(2.0**-4 * (y.abs() + off), 2.0**-10 * s) * (1 + 2 * U)
    near = (q.double() * s - y).abs() <= off + half  # (false where a value is NaN)
    assert near.all(), (~near).nonzero()[:4].tolist()
