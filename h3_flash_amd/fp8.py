"""Linear layers of a DiT block in 8 bits (HIP, gfx950).

A matrix in 8 bits is a pair: its values as ``torch.float8_e4m3fn`` and its scales as
``torch.float8_e8m0fnu``, powers of two, which the matrix cores apply themselves.
Activations have a scale for every row and 128 columns (:func:`quantize_fp8`), weights
one for every block of 128 x 128 (:func:`quantize_fp8_weight`, once, when a model is
loaded). A scale is the smallest power of two by which no value of its group passes
448, e4m3's largest; a group that holds a value that is not finite is NaN throughout.

:func:`fused_linear_fp8` is :func:`h3_flash_amd.fused_linear` on such pairs. Between
the steps of a block nothing need be rounded to bf16 first: the norms before a branch
end in 8 bits (:func:`h3_flash_amd.fusions.fused_rmsnorm_modulate_fp8`,
:func:`h3_flash_amd.fusions.fused_residual_gate_rmsnorm_modulate_fp8`), and the MLP's up
projection does with ``quantize=True``::

    hidden, q, q_scale = fused_residual_gate_rmsnorm_modulate_fp8(residual, branch, ...)
    q, q_scale = fused_linear_fp8(q, up, up_scale, x_scale=q_scale, activation="silu", gated=True, quantize=True)
    y = fused_linear_fp8(q, down, down_scale, x_scale=q_scale, residual=hidden, gate=gate, index=index)
"""

from __future__ import annotations

import torch

from . import _ext
from .fusions import _aligned_rows, _dtype, _empty, _fp8_scales, _index, _index_args, _operand, _tables, _vector

__all__ = ["fused_linear_fp8", "quantize_fp8", "quantize_fp8_weight"]

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_BF16_F32 = {torch.bfloat16: (_ext.H3A_DTYPE_BF16, 2), torch.float32: (_ext.H3A_DTYPE_F32, 4)}


def _groups(n: int) -> int:
    return (n + 127) // 128


def _held_rows(x: torch.Tensor, columns: int) -> tuple[torch.Tensor, int, int]:
    """The tensor that holds x's rows as 16-byte aligned ones, their number and stride."""

    size = x.element_size()
    if x.is_contiguous() and columns * size % 16 == 0 and x.data_ptr() % 16 == 0:
        return x, x.numel() // columns, columns
    x = x if x.dim() == 2 else x.reshape(-1, columns)
    stride = x.stride(0)
    if x.stride(1) != 1 or stride < columns or stride * size % 16 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        stride = columns
    return x, x.shape[0], stride


def _held_scales(scale: torch.Tensor, rows: int, columns: int) -> tuple[torch.Tensor, int]:
    """Rows of scales that start at multiples of 16 bytes, whole 16 bytes of each in
    their storage (else a copy), and their stride."""

    pitch = (columns + 15) // 16 * 16
    flat = scale if scale.dim() == 2 else scale.reshape(-1, columns)
    stride = flat.stride(0) if rows > 1 else pitch
    if (
        (flat.stride(1) == 1 or columns == 1)
        and stride % 16 == 0
        and stride >= columns
        and flat.data_ptr() % 16 == 0
        and flat.storage_offset() + rows * stride <= flat.untyped_storage().nbytes()
    ):
        return flat, stride
    held = torch.zeros((rows, pitch), dtype=torch.uint8, device=scale.device)
    held[:, :columns] = flat.view(torch.uint8)
    return held, pitch


def _quantize(x: torch.Tensor, name: str, scale_rows: tuple[int, ...], block_rows: int, parts: int):
    if x.dtype not in _BF16_F32:
        raise TypeError(f"{name} must be bfloat16 or float32, got {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be on a ROCm device, got {x.device}")
    columns = x.shape[-1]
    if columns == 0 or columns % 16:
        raise ValueError(f"{name}'s last dimension must be a positive multiple of 16, got {columns}")
    held, rows, stride = _held_rows(x, columns)
    q = _empty(x.shape, E4M3, x.device)
    scale, pitch = _fp8_scales(scale_rows, columns, x.device)
    if rows:
        _ext.quantize_fp8.run(
            x.device, _ext.ABI_VERSION, held.data_ptr(), _BF16_F32[x.dtype][0], q.data_ptr(), scale.data_ptr(), rows, columns,
            block_rows, parts, stride, columns, pitch,
        )
    return q, scale


def quantize_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)``: rows of activations in 8 bits.

    ``x``: (..., k) bf16 or fp32, ``k`` a multiple of 16. ``q``: (..., k) e4m3,
    contiguous; ``scale``: (..., ceil(k / 128)) e8m0, whose rows start at multiples of
    16 bytes (a view of a wider tensor unless ceil(k / 128) is one). ``x`` is about
    ``q * scale``, each value off by at most half a step of e4m3 (2^-4 of it, or 2^-10
    of the scale where that is more)."""

    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    return _quantize(x, "x", x.shape[:-1], 1, 1)


def quantize_fp8_weight(weight: torch.Tensor, *, gated: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)``: a weight in 8 bits, for :func:`fused_linear_fp8`.

    ``weight``: (n, k) bf16 or fp32, ``k`` a multiple of 16, the ``nn.Linear`` layout;
    ``scale``: (ceil(n / 128), ceil(k / 128)) e8m0. With ``gated`` the weight holds 2 n
    rows, values then gates, and ``scale`` the blocks of the n value rows, then those of
    the n gate rows."""

    if weight.dim() != 2:
        raise ValueError(f"weight must be 2-D, got {tuple(weight.shape)}")
    rows = weight.shape[0]
    if gated and rows % 2:
        raise ValueError(f"a gated weight needs an even number of rows, got {rows}")
    parts = 2 if gated else 1
    return _quantize(weight, "weight", (parts * _groups(rows // parts),), 128, parts)


def fused_linear_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    x_scale: torch.Tensor | None = None,
    activation: str | None = None,
    gated: bool = False,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    index: torch.Tensor | None = None,
    quantize: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``residual + gate[t] * act(x @ weight^T + bias)`` of operands in 8 bits, with
    ``t = index[row % len(index)]`` (clamped to the table); terms not given are left out.

    ``weight``, ``weight_scale``: :func:`quantize_fp8_weight`'s, (n, k) (with ``gated``
    as given there). ``x``: (..., k) e4m3 with its ``x_scale`` (..., ceil(k / 128)) e8m0,
    as :func:`quantize_fp8` and the norms give them; or bf16 without one, which is
    rounded to 8 bits in the same way first. ``bias``, ``activation``, ``gated``,
    ``residual``, ``gate``, ``index`` and ``out`` as for
    :func:`h3_flash_amd.fused_linear`. ``quantize=True``: the fp32 result is not rounded
    to bf16 but to 8 bits, and ``(q, scale)`` is returned, as from :func:`quantize_fp8`
    (without ``out``). ``k`` is a multiple of 16, ``n`` of 8, with ``quantize`` of 16.

    The matrix cores line up eight neighbouring products of k to the largest of them, 13
    bits kept below it, and accumulate those sums in fp32: they are some 3e-4 of the
    result's norm off. A bf16 result's rounding (1.7e-3) covers that; with ``quantize`` a
    value next to the middle of two e4m3 values may become the other one, 0.3 to 0.9% of
    the norm in all, where the rounding itself is 2.6%.
    With ``quantize`` a reduction is not cut into pieces: over a long ``k`` with a small
    result (up to some hundred tokens, ``n`` of a few thousand) :func:`quantize_fp8` of the
    bf16 result is the faster way.
    """

    if weight.dim() != 2 or weight.dtype != E4M3:
        raise TypeError(f"weight must be a 2-D float8_e4m3fn tensor, got {weight.dtype} {tuple(weight.shape)}")
    if activation not in _ext.ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_ext.ACTIVATIONS)}, got {activation!r}")
    rows, k = weight.shape
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} are incompatible")
    if gated and rows % 2:
        raise ValueError(f"a gated product needs an even number of weight rows, got {rows}")
    n = rows // 2 if gated else rows
    n_step = 16 if quantize else 8
    if k % 16 or n % n_step or k == 0 or n == 0:
        raise ValueError(f"k must be a positive multiple of 16 and n of {n_step}, got {k} and {n}")
    if not x.is_cuda:
        raise RuntimeError(f"x must be on a ROCm device, got {x.device}")
    device, kb = x.device, _groups(k)
    blocks = (2 if gated else 1) * _groups(n)
    if weight_scale.dtype != E8M0:
        raise TypeError(f"weight_scale must be float8_e8m0fnu, got {weight_scale.dtype}")
    if weight_scale.shape != (blocks, kb):
        raise ValueError(f"weight_scale must be {(blocks, kb)}, got {tuple(weight_scale.shape)}")
    if weight.device != device or weight_scale.device != device:
        raise ValueError(f"x, weight and weight_scale must be on one device, got {device}, {weight.device} and {weight_scale.device}")
    shape = (*x.shape[:-1], n)
    if x_scale is None:
        if x.dtype != torch.bfloat16:
            raise TypeError(f"x must be bfloat16, or float8_e4m3fn with an x_scale, got {x.dtype}")
        flat, m, x_stride = _operand(x, "x", k)
        x_args, xs_args = (flat.data_ptr(), _ext.H3A_DTYPE_BF16, 0), (x_stride, 0)
    else:
        if x.dtype != E4M3 or x_scale.dtype != E8M0:
            raise TypeError(f"x and x_scale must be float8_e4m3fn and float8_e8m0fnu, got {x.dtype} and {x_scale.dtype}")
        if x_scale.shape != (*x.shape[:-1], kb):
            raise ValueError(f"x_scale must be {(*x.shape[:-1], kb)}, got {tuple(x_scale.shape)}")
        if x_scale.device != device:
            raise ValueError(f"x and x_scale must be on one device, got {device} and {x_scale.device}")
        flat, m, x_stride = _held_rows(x, k)
        x_scale, xs_stride = _held_scales(x_scale, m, kb)
        x_args, xs_args = (flat.data_ptr(), _ext.H3A_DTYPE_F8E4M3, x_scale.data_ptr()), (x_stride, xs_stride)
    weight = _aligned_rows(weight)
    weight_scale, ws_stride = _held_scales(weight_scale, blocks, kb)
    if bias is not None:
        bias = _vector(bias, rows, device, "bias")
        bias = bias if bias.data_ptr() % 16 == 0 else bias.clone()
    residual_stride = 0
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual must be {shape}, got {tuple(residual.shape)}")
        if residual.device != device:
            raise ValueError(f"x and residual must be on one device, got {device} and {residual.device}")
        residual, _, residual_stride = _operand(residual, "residual", n)
    gate_args = (0, _ext.H3A_DTYPE_BF16, 0, 0, 0, _ext.H3A_DTYPE_I64, 0)
    if gate is not None:
        if index is None:
            raise ValueError("gate needs an index")
        (gate,) = _tables([gate], n, device)
        gate, index = _aligned_rows(gate), _index(index, device)
        at, index_dtype, n_index = _index_args(index)
        gate_args = (gate.data_ptr(), _dtype(gate), gate.stride(0), gate.shape[0], at, index_dtype, n_index)
    y_stride, y_scale, ys_stride = n, None, 0
    if quantize:
        if out is not None:
            raise ValueError("quantize and out exclude each other")
        y = out = _empty(shape, E4M3, device)
        y_scale, ys_stride = _fp8_scales(shape[:-1], n, device)
    elif out is None:
        y = out = _empty(shape, torch.bfloat16, device)
    else:
        if out.shape != shape or out.dtype != torch.bfloat16 or out.device != device:
            raise ValueError(f"out must be a bf16 {shape} tensor on {device}")
        y = out.view(-1, n) if m else out.new_empty((0, n))
        if m and (y.stride(1) != 1 or y.stride(0) % 8 or y.stride(0) < n or y.data_ptr() % 16):
            raise ValueError("out must have contiguous, 16-byte aligned rows")
        y_stride = y.stride(0)
    if m:
        args = (
            _ext.ABI_VERSION, *x_args, weight.data_ptr(), weight_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
            _ext.H3A_DTYPE_BF16 if bias is None else _dtype(bias), 0 if residual is None else residual.data_ptr(), *gate_args,
            y.data_ptr(), _ext.H3A_DTYPE_F8E4M3 if quantize else _ext.H3A_DTYPE_BF16, y_scale.data_ptr() if quantize else 0,
            m, k, n, *xs_args, weight.stride(0), ws_stride, residual_stride, y_stride, ys_stride,
            _ext.ACTIVATIONS[activation], int(gated),
        )
        rc = _ext.linear_fp8(device, *args, 0, _ext.H3A_WORKSPACE_ASK)
        if rc == _ext.H3A_NEED_WORKSPACE:
            need = _ext.linear_fp8_workspace_size(device, *args, 0, 0)
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            rc = _ext.linear_fp8(device, *args, workspace.data_ptr(), need)
        if rc != _ext.H3A_OK:
            _ext.check(_ext.load_library(), rc)
    return (out, y_scale) if quantize else out
