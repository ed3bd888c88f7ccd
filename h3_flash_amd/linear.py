"""Matrix products of a DiT block with what follows them in the epilogue (HIP,
gfx950): bias, activation or gated activation, modulation gate and residual.

One launch takes the place of a linear layer and the row kernels after it: the
MLP's up projection with :func:`h3_flash_amd.fusions.fused_swiglu` (``gated=True,
activation="silu"``: the same halves, values first), its down projection with the
gated residual of the block, and the projection of a timestep embedding to
modulation rows, whose few tokens run on a form that streams the weights once.
Everything between the operands and the result is computed in fp32 and rounded to
bf16 once (the separate steps round the product, too).
"""

from __future__ import annotations

import torch

from . import _ext
from .fusions import _dtype, _index, _index_args, _row_span, _rows, _tables, _vector

__all__ = ["fused_linear"]


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """Rows of 16-byte chunks, as the launch reads them (else a copy)."""

    row, column = t.stride()
    if column == 1 and row * t.element_size() % 16 == 0 and row >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _operand(x: torch.Tensor, name: str, columns: int) -> tuple[torch.Tensor, int, int]:
    """Rows of 16-byte chunks: the tensor that holds them, their number and stride."""

    held, rows, stride = _row_span(x, name, columns)
    if stride % 8 or stride < columns or held.data_ptr() % 16:
        held = _aligned_rows(_rows(held, name, columns))
        stride = held.stride(0)
    return held, rows, stride


def fused_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    gated: bool = False,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    index: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``residual + gate[t] * act(x @ weight^T + bias)`` with ``t = index[row %
    len(index)]`` (clamped to the table); terms not given are left out.

    ``x``: (..., k) bf16; ``weight``: (n, k) bf16, the ``nn.Linear`` layout;
    ``bias``: (n,) and ``gate``: (rows, n), each bf16 or fp32; ``residual`` and
    ``out``: (..., n) bf16. ``activation``: None, "silu", "gelu", "gelu_tanh" or
    "relu". With ``gated`` the weight (and bias) hold 2 n rows, values then gates,
    and the product is ``value * act(gate)``. ``k`` and ``n`` are multiples of 8.
    ``out`` may be the residual itself and overlaps no other operand (ValueError).
    """

    if weight.dim() != 2 or weight.dtype != torch.bfloat16:
        raise TypeError(f"weight must be a 2-D bfloat16 tensor, got {weight.dtype} {tuple(weight.shape)}")
    if activation not in _ext.ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_ext.ACTIVATIONS)}, got {activation!r}")
    rows, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} are incompatible")
    if gated and rows % 2:
        raise ValueError(f"a gated product needs an even number of weight rows, got {rows}")
    n = rows // 2 if gated else rows
    if k % 8 or n % 8 or k == 0 or n == 0:
        raise ValueError(f"k and n must be positive multiples of 8, got {k} and {n}")
    flat, m, x_stride = _operand(x, "x", k)
    device = x.device
    if weight.device != device:
        raise ValueError(f"x and weight must be on one device, got {device} and {weight.device}")
    weight = _aligned_rows(weight)
    if bias is not None:
        bias = _vector(bias, rows, device, "bias")
        bias = bias if bias.data_ptr() % 16 == 0 else bias.clone()
    shape, residual_stride = (*x.shape[:-1], n), 0
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
    y_stride = n
    if out is None:
        y = out = flat.new_empty(shape)
    else:
        if out.shape != shape or out.dtype != torch.bfloat16 or out.device != device:
            raise ValueError(f"out must be a bf16 {shape} tensor on {device}")
        y = out.view(-1, n) if m else out.new_empty((0, n))
        if m and (y.stride(1) != 1 or y.stride(0) % 8 or y.stride(0) < n or y.data_ptr() % 16):
            raise ValueError("out must have contiguous, 16-byte aligned rows")
        y_stride = y.stride(0)
    if m:
        args = (
            _ext.ABI_VERSION, flat.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(),
            _ext.H3A_DTYPE_BF16 if bias is None else _dtype(bias), 0 if residual is None else residual.data_ptr(), *gate_args,
            y.data_ptr(), m, k, n, x_stride, weight.stride(0), residual_stride, y_stride,
            _ext.ACTIVATIONS[activation], int(gated),
        )
        rc = _ext.linear(device, *args, 0, _ext.H3A_WORKSPACE_ASK)
        if rc == _ext.H3A_NEED_WORKSPACE:
            need = _ext.linear_workspace_size(device, *args, 0, 0)
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            rc = _ext.linear(device, *args, workspace.data_ptr(), need)
        if rc != _ext.H3A_OK:
            _ext.check(_ext.load_library(), rc)
    return out
