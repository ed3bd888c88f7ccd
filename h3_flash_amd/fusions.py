"""Row-wise fusions of the MiniMax H3 DiT block on MI355X (HIP, gfx950).

Same function names, arguments and return values as the reference's Triton
wrappers (src/h3_flash/runtime/kernels/fusions.py):

* :func:`fused_rmsnorm_modulate` (fusions.py:194-215)
* :func:`fused_residual_gate_rmsnorm_modulate` (fusions.py:218-248)
* :func:`fused_swiglu` (fusions.py:251-265)
* :func:`fused_qknorm_rope` (fusions.py:268-293), from :mod:`h3_flash_amd.prologue`

and, for blocks that also normalise what a branch returns,
:func:`fused_rmsnorm_residual_gate_rmsnorm_modulate`, which the reference lacks,
and, with their result in 8 bits for :func:`h3_flash_amd.fused_linear_fp8`,
:func:`fused_rmsnorm_modulate_fp8` and :func:`fused_residual_gate_rmsnorm_modulate_fp8`.

Activations are bf16 (the dtype the H3 block runs in); weights and
modulation tables may be bf16 or fp32, table indices int32 or int64. Table
indices outside the table are clamped to it (the reference reads out of
bounds there). Every call is one HIP launch on the current stream.
"""

from __future__ import annotations

import torch

from . import _ext
from .prologue import fused_qknorm_rope

__all__ = [
    "fused_qknorm_rope",
    "fused_residual_gate_rmsnorm_modulate",
    "fused_residual_gate_rmsnorm_modulate_fp8",
    "fused_rmsnorm_modulate",
    "fused_rmsnorm_modulate_fp8",
    "fused_rmsnorm_residual_gate_rmsnorm_modulate",
    "fused_swiglu",
]


def _rows(x: torch.Tensor, name: str, columns: int) -> torch.Tensor:
    """(N, columns) bf16 device view with a contiguous last dimension."""

    if x.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be on a ROCm device, got {x.device}")
    flat = x if x.dim() == 2 else x.reshape(-1, columns)
    return flat if flat.stride(1) == 1 else flat.contiguous()


def _row_span(x: torch.Tensor, name: str, columns: int) -> tuple[torch.Tensor, int, int]:
    """The tensor that holds x's rows as :func:`_rows` gives them, their number and
    stride (a contiguous x as it is: no view is made of it)."""

    if x.is_contiguous() and x.dtype == torch.bfloat16 and x.is_cuda and columns:
        return x, x.numel() // columns, columns
    flat = _rows(x, name, columns)
    return flat, flat.shape[0], flat.stride(0)


def _vector(t: torch.Tensor, columns: int, device: torch.device, name: str) -> torch.Tensor:
    if t.shape != (columns,):
        if t.shape[-1] != columns or t.numel() != columns:
            raise ValueError(f"{name} must have {columns} elements, got shape {tuple(t.shape)}")
        t = t.reshape(columns)
    if t.device != device:
        t = t.to(device)
    if t.dtype not in (torch.bfloat16, torch.float32):
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _tables(tables: list[torch.Tensor], columns: int, device: torch.device) -> list[torch.Tensor]:
    out, dtype = [], torch.bfloat16
    for t in tables:
        if t.dim() != 2 or t.shape[1] != columns:
            raise ValueError(f"modulation tables must be (rows, {columns}), got {tuple(t.shape)}")
        if t.dtype != torch.bfloat16:
            dtype = torch.float32
        out.append(t if t.device == device else t.to(device))
    # _row_addressable (fusions.py:190-191): the last dimension must be
    # contiguous; broadcast rows (a row stride under the row, e.g. expand())
    # are written out, since the launch takes one row stride per table
    for i, t in enumerate(out):
        if t.dtype != dtype:
            t = out[i] = t.to(dtype)
        row, column = t.stride()
        if column != 1 or row < columns:
            out[i] = t.contiguous()
    return out


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """Rows of 16-byte chunks, as the launch reads them (else a copy)."""

    row, column = t.stride()
    if column == 1 and row * t.element_size() % 16 == 0 and row >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _empty(shape: tuple[int, ...], dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A contiguous empty tensor (of a matrix by its strides: half the call's time)."""

    if len(shape) == 2:
        return torch.empty_strided(shape, (max(shape[1], 1), 1), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _fp8_scales(lead: tuple[int, ...], columns: int, device: torch.device) -> tuple[torch.Tensor, int]:
    """An empty (*lead, ceil(columns / 128)) tensor of e8m0 scales whose rows start at
    multiples of 16 bytes, and their stride."""

    groups = (columns + 127) // 128
    pitch = (groups + 15) // 16 * 16
    scale = _empty((*lead, pitch), torch.float8_e8m0fnu, device)
    if pitch == groups:
        return scale, pitch
    return (scale.as_strided((lead[0], groups), (pitch, 1)) if len(lead) == 1 else scale[..., :groups]), pitch


def _operand(x: torch.Tensor, name: str, columns: int) -> tuple[torch.Tensor, int, int]:
    """:func:`_row_span` in rows of 16-byte chunks, as the launch reads them (else a copy)."""

    held, rows, stride = _row_span(x, name, columns)
    if stride % 8 or stride < columns or held.data_ptr() % 16:
        held = _aligned_rows(_rows(held, name, columns))
        stride = held.stride(0)
    return held, rows, stride


def _index(index: torch.Tensor, device: torch.device) -> torch.Tensor:
    if index.dim() != 1:
        index = index.reshape(-1)
    if index.device != device:
        index = index.to(device)
    if index.numel() == 0:
        raise ValueError("index must not be empty")
    if index.dtype not in (torch.int32, torch.int64):
        index = index.long()
    return index if index.is_contiguous() else index.contiguous()


def _dtype(t: torch.Tensor) -> int:
    return _ext.H3A_DTYPE_F32 if t.dtype == torch.float32 else _ext.H3A_DTYPE_BF16


def _index_args(index: torch.Tensor) -> tuple[int, int, int]:
    return index.data_ptr(), _ext.H3A_DTYPE_I64 if index.dtype == torch.int64 else _ext.H3A_DTYPE_I32, index.numel()


def fused_rmsnorm_modulate(x, weight, scale, shift, index, eps):
    """RMSNorm over the last dimension, times ``weight``, then
    ``* (1 + scale[t]) + shift[t]`` with ``t = index[row % len(index)]``."""

    columns = x.shape[-1]
    flat = _rows(x, "x", columns)
    weight = _vector(weight, columns, x.device, "weight")
    scale, shift = _tables([scale, shift], columns, x.device)
    index = _index(index, x.device)
    output = flat.new_empty((flat.shape[0], columns))
    _ext.rmsnorm_modulate.run(
        x.device, _ext.ABI_VERSION, flat.data_ptr(), output.data_ptr(), weight.data_ptr(), _dtype(weight),
        scale.data_ptr(), shift.data_ptr(), _dtype(scale), scale.stride(0), shift.stride(0),
        min(scale.shape[0], shift.shape[0]), *_index_args(index), flat.shape[0], columns,
        flat.stride(0), output.stride(0), float(eps),
    )
    return output.view(x.shape)


def fused_residual_gate_rmsnorm_modulate(residual, branch, gate, weight, scale, shift, index, eps):
    """``hidden = residual + gate[t] * branch``, then RMSNorm(hidden) * weight
    * (1 + scale[t]) + shift[t]; returns ``(hidden, normed)``."""

    columns = residual.shape[-1]
    if branch.shape != residual.shape:
        raise ValueError(f"residual {tuple(residual.shape)} and branch {tuple(branch.shape)} differ")
    residual_flat = _rows(residual, "residual", columns)
    branch_flat = _rows(branch, "branch", columns)
    if branch.device != residual.device:
        raise ValueError(f"residual and branch must be on one device, got {residual.device} and {branch.device}")
    weight = _vector(weight, columns, residual.device, "weight")
    gate, scale, shift = _tables([gate, scale, shift], columns, residual.device)
    index = _index(index, residual.device)
    rows = residual_flat.shape[0]
    hidden, normed = residual_flat.new_empty((rows, columns)), residual_flat.new_empty((rows, columns))
    _ext.residual_gate_rmsnorm_modulate.run(
        residual.device, _ext.ABI_VERSION, residual_flat.data_ptr(), branch_flat.data_ptr(), hidden.data_ptr(),
        normed.data_ptr(), weight.data_ptr(), _dtype(weight), gate.data_ptr(), scale.data_ptr(), shift.data_ptr(),
        _dtype(gate), gate.stride(0), scale.stride(0), shift.stride(0),
        min(gate.shape[0], scale.shape[0], shift.shape[0]), *_index_args(index), residual_flat.shape[0], columns,
        residual_flat.stride(0), branch_flat.stride(0), hidden.stride(0), normed.stride(0), float(eps),
    )
    return hidden.view(residual.shape), normed.view(residual.shape)


def fused_rmsnorm_residual_gate_rmsnorm_modulate(
    residual, branch, branch_weight, gate, weight, scale, shift, index, eps, *, residual_scale=1.0
):
    """``hidden = residual_scale * residual + gate[t] * RMSNorm(branch) *
    branch_weight``, then ``RMSNorm(hidden) * weight * (1 + scale[t]) +
    shift[t]``; returns ``(hidden, normed)``.

    ``gate=None`` leaves the gate out. ``weight=None`` (with ``scale`` and
    ``shift`` None) ends at the hidden state, as after a model's last block, and
    returns ``(hidden, None)``; ``index`` may be None when no table is given."""

    shape = residual.shape
    columns = shape[-1]
    if branch.shape != shape:
        raise ValueError(f"residual {tuple(shape)} and branch {tuple(branch.shape)} differ")
    norm = weight is not None
    if norm != (scale is not None) or norm != (shift is not None):
        raise ValueError("weight, scale and shift go together: give all three or none")
    device = residual.device
    rows_r, n_rows, stride_r = _row_span(residual, "residual", columns)
    rows_b, _, stride_b = _row_span(branch, "branch", columns)
    if branch.device != device:
        raise ValueError(f"residual and branch must be on one device, got {device} and {branch.device}")
    branch_weight = _vector(branch_weight, columns, device, "branch_weight")
    w_ptr = 0
    if norm:
        weight = _vector(weight, columns, device, "weight")
        if weight.dtype != branch_weight.dtype:  # one dtype for both
            weight, branch_weight = weight.float(), branch_weight.float()
        w_ptr = weight.data_ptr()
    gate_ptr = gate_stride = scale_ptr = scale_stride = shift_ptr = shift_stride = table_rows = 0
    table_dtype, index_args = _ext.H3A_DTYPE_BF16, (0, _ext.H3A_DTYPE_I64, 0)
    if norm or gate is not None:
        if index is None:
            raise ValueError("gate, scale and shift need an index")
        tables = _tables([t for t in (gate, scale, shift) if t is not None], columns, device)
        table_dtype, table_rows = _dtype(tables[0]), min([t.shape[0] for t in tables])
        if gate is not None:
            gate_ptr, gate_stride = tables[0].data_ptr(), tables[0].stride(0)
        if norm:
            scale, shift = tables[-2:]
            scale_ptr, scale_stride, shift_ptr, shift_stride = scale.data_ptr(), scale.stride(0), shift.data_ptr(), shift.stride(0)
        index = _index(index, device)
        index_args = _index_args(index)
    hidden = torch.empty_like(residual, memory_format=torch.contiguous_format)
    normed = torch.empty_like(hidden) if norm else None
    if columns:
        _ext.rmsnorm_residual_gate_rmsnorm_modulate.run(
            device, _ext.ABI_VERSION, rows_r.data_ptr(), rows_b.data_ptr(), hidden.data_ptr(),
            normed.data_ptr() if norm else 0, branch_weight.data_ptr(), w_ptr, _dtype(branch_weight), gate_ptr, scale_ptr,
            shift_ptr, table_dtype, gate_stride, scale_stride, shift_stride, table_rows, *index_args, n_rows, columns,
            stride_r, stride_b, columns, columns, float(residual_scale), float(eps),
        )
    return hidden, normed


def _norm_fp8_args(weight, tables, index, columns, device):
    """The norm weight, the modulation tables in 16-byte aligned rows, and the index."""

    if columns == 0 or columns % 16:
        raise ValueError(f"the last dimension must be a positive multiple of 16, got {columns}")
    weight = _vector(weight, columns, device, "weight")
    weight = weight if weight.data_ptr() % 16 == 0 else weight.clone()
    tables = [_aligned_rows(t) for t in _tables(tables, columns, device)]
    return weight, tables, _index(index, device)


def fused_rmsnorm_modulate_fp8(x, weight, scale, shift, index, eps):
    """:func:`fused_rmsnorm_modulate` with its result in 8 bits, rounded from fp32:
    returns ``(q, q_scale)`` as :func:`h3_flash_amd.quantize_fp8` does, for
    :func:`h3_flash_amd.fused_linear_fp8`. The last dimension is a multiple of 16, at
    most 16,384."""

    columns = x.shape[-1]
    device = x.device
    held, rows, stride = _operand(x, "x", columns)
    weight, tables, index = _norm_fp8_args(weight, [scale, shift], index, columns, device)
    scale, shift = tables
    q = _empty(x.shape, torch.float8_e4m3fn, device)
    q_scale, pitch = _fp8_scales(x.shape[:-1], columns, device)
    _ext.rmsnorm_modulate_fp8.run(
        device, _ext.ABI_VERSION, held.data_ptr(), q.data_ptr(), q_scale.data_ptr(), weight.data_ptr(), _dtype(weight),
        scale.data_ptr(), shift.data_ptr(), _dtype(scale), scale.stride(0), shift.stride(0),
        min(scale.shape[0], shift.shape[0]), *_index_args(index), rows, columns, stride, columns, pitch, float(eps),
    )
    return q, q_scale


def fused_residual_gate_rmsnorm_modulate_fp8(residual, branch, gate, weight, scale, shift, index, eps):
    """:func:`fused_residual_gate_rmsnorm_modulate` with its normed rows in 8 bits:
    returns ``(hidden, q, q_scale)``, ``hidden`` in bf16, the others as from
    :func:`fused_rmsnorm_modulate_fp8`."""

    columns = residual.shape[-1]
    device = residual.device
    if branch.shape != residual.shape:
        raise ValueError(f"residual {tuple(residual.shape)} and branch {tuple(branch.shape)} differ")
    rows_r, rows, stride_r = _operand(residual, "residual", columns)
    rows_b, _, stride_b = _operand(branch, "branch", columns)
    if branch.device != device:
        raise ValueError(f"residual and branch must be on one device, got {device} and {branch.device}")
    weight, tables, index = _norm_fp8_args(weight, [gate, scale, shift], index, columns, device)
    gate, scale, shift = tables
    hidden, q = _empty(residual.shape, torch.bfloat16, device), _empty(residual.shape, torch.float8_e4m3fn, device)
    q_scale, pitch = _fp8_scales(residual.shape[:-1], columns, device)
    _ext.residual_gate_rmsnorm_modulate_fp8.run(
        device, _ext.ABI_VERSION, rows_r.data_ptr(), rows_b.data_ptr(), hidden.data_ptr(), q.data_ptr(), q_scale.data_ptr(),
        weight.data_ptr(), _dtype(weight), gate.data_ptr(), scale.data_ptr(), shift.data_ptr(), _dtype(gate), gate.stride(0),
        scale.stride(0), shift.stride(0), min(gate.shape[0], scale.shape[0], shift.shape[0]), *_index_args(index), rows, columns,
        stride_r, stride_b, columns, columns, pitch, float(eps),
    )
    return hidden, q, q_scale


def fused_swiglu(x):
    """``value * silu(gate)`` with ``value, gate = x.chunk(2, -1)``."""

    if x.shape[-1] % 2:
        raise ValueError(f"swiglu needs an even last dimension, got {x.shape[-1]}")
    columns = x.shape[-1] // 2
    flat = _rows(x, "x", x.shape[-1])
    output = flat.new_empty((flat.shape[0], columns))
    _ext.swiglu.run(
        x.device, _ext.ABI_VERSION, flat.data_ptr(), output.data_ptr(), flat.shape[0], columns,
        flat.stride(0), output.stride(0),
    )
    return output.view(*x.shape[:-1], columns)
