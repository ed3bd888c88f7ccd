"""Attention over selected key blocks on MI355X (HIP, gfx950).

:func:`select_key_blocks` scores the 64-key blocks of a sequence for every block
of 256 queries by the product of their means and names the best ones;
:func:`sparse_attn_func` attends to the blocks that such lists name.
:class:`BlockSparseKernel` is both behind the call form of
:func:`h3_flash_amd.flash_attn_func`, for
``DenseMiniMaxH3Processor(kernel=BlockSparseKernel(keep=0.2))``. The reference's
attention is dense; these are for models that were made or tuned for block
sparsity.
"""

from __future__ import annotations

import math

import torch

from . import _ext
from .attention import HEAD_DIM, _as_kernel_operand, _strides3

__all__ = ["BLOCK_K", "BLOCK_Q", "BlockSparseKernel", "select_key_blocks", "sparse_attn_func"]

BLOCK_Q = _ext.H3A_BLOCK_Q  # query rows that share a list
BLOCK_K = _ext.H3A_BLOCK_K  # keys of a listed block


def _blocks(n: int, size: int) -> int:
    return -(-n // size)


def _select_workspace(heads: int, nq: int, nk: int) -> int:
    """What h3a_block_select_workspace_size returns, without the call: the means and
    scores, each from a 256-byte boundary on (the tests hold the two equal)."""

    return sum(-(-heads * n // 256) * 256 for n in (nq * 512, nk * 512, nq * nk * 4))


def _check_pair(q: torch.Tensor, k: torch.Tensor) -> None:
    if q.shape[3] != HEAD_DIM:
        raise ValueError(f"head_dim must be {HEAD_DIM}, got {q.shape[3]}")
    if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} are incompatible")
    if k.shape[2] != q.shape[2]:
        raise RuntimeError("H3 sparse HIP attention does not support grouped-query attention")
    if k.device != q.device:
        raise ValueError("q, k and v must be on the same device")


def select_key_blocks(
    q: torch.Tensor, k: torch.Tensor, topk: int, *, always: torch.Tensor | None = None
) -> torch.Tensor:
    """The ``min(topk, nk)`` key blocks of each query block with the largest
    ``<mean of its queries, mean of the block's keys>``: int32 (B, H, nq, topk),
    ascending, with ``nq`` blocks of 256 query rows and ``nk`` of 64 keys (the
    last of either may be shorter).

    ``q``, ``k``: (B, S, H, 128) bf16, as for :func:`flash_attn_func`. ``always``:
    a truth value per key block; the marked blocks (those of a text prefix, say)
    come before all others, the lowest first. Sums are taken in 64 bits; equal
    scores go to the lowest index, NaN counts as -inf.
    """

    q, k = _as_kernel_operand(q, "q"), _as_kernel_operand(k, "k")
    _check_pair(q, k)
    if topk < 1:
        raise ValueError(f"topk must be positive, got {topk}")
    B, Sq, H, D = q.shape
    nq, nk = _blocks(Sq, BLOCK_Q), _blocks(k.shape[1], BLOCK_K)
    device = q.device
    if always is not None:
        if always.shape != (nk,):
            raise ValueError(f"always must have one value for each of the {nk} key blocks, got {tuple(always.shape)}")
        always = always.to(device=device, dtype=torch.bool).contiguous()
    topk = min(int(topk), nk)
    index = torch.empty((B, H, nq, topk), dtype=torch.int32, device=device)
    if index.numel() == 0:
        return index
    args = (
        _ext.ABI_VERSION, q.data_ptr(), k.data_ptr(), 0 if always is None else always.data_ptr(), index.data_ptr(),
        B, H, Sq, k.shape[1], D, *_strides3(q), *_strides3(k), topk,
    )
    need = _select_workspace(B * H, nq, nk)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _ext.block_select.run(device, *args, workspace.data_ptr(), need)
    return index


def sparse_attn_func(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    block_index: torch.Tensor,
    block_count: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    *,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of each block of 256 query rows to the 64-key blocks that its
    list names; returns ``(out, lse)`` as :func:`flash_attn_func` does.

    ``q``: (B, Sq, H, 128), ``k``/``v``: (B, Sk, H, 128), bf16. ``block_index``:
    int32 (B, H, nq, n), ``block_count`` (B, H, nq) the number of its entries used
    (default: all; clamped to [0, n]). Entries may come in any order; a block
    named twice counts twice, as two keys would; entries outside [0, nk) name
    nothing. A row without keys has ``out`` 0 and ``lse`` -inf. Lists hold at most
    7,168 entries. ``out`` and ``lse``, where given, overlap no input.

    Scores, sums and ``lse`` are fp32; the softmax weights are rounded to bf16 for
    the product with ``v`` (by at most 2^-8 of each), as in
    :func:`flash_attn_func`, and the result once more.
    """

    q, k, v = _as_kernel_operand(q, "q"), _as_kernel_operand(k, "k"), _as_kernel_operand(v, "v")
    _check_pair(q, k)
    if k.shape != v.shape:
        raise ValueError(f"k and v shapes differ: {tuple(k.shape)} vs {tuple(v.shape)}")
    device = q.device
    if v.device != device:
        raise ValueError("q, k and v must be on the same device")
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    nq = _blocks(Sq, BLOCK_Q)
    if block_index.dim() != 4 or block_index.shape[:3] != (B, H, nq):
        raise ValueError(f"block_index must be ({B}, {H}, {nq}, n), got {tuple(block_index.shape)}")
    if block_index.dtype != torch.int32 or block_index.device != device:
        raise ValueError(f"block_index must be an int32 tensor on {device}")
    if block_index.stride(3) != 1:
        block_index = block_index.contiguous()
    counts = (0, 0, 0, 0)
    if block_count is not None:
        if block_count.shape != (B, H, nq) or block_count.dtype != torch.int32 or block_count.device != device:
            raise ValueError(f"block_count must be an int32 ({B}, {H}, {nq}) tensor on {device}")
        counts = (block_count.data_ptr(), *block_count.stride())
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    if out is None:
        out = q.new_empty((B, Sq, H, D))
    elif out.shape != (B, Sq, H, D) or out.dtype != torch.bfloat16 or out.stride(-1) != 1 or out.device != device:
        raise ValueError(f"out must be a bf16 (B, Sq, H, 128) tensor on {device} with a contiguous last dim")
    if lse is None:
        lse = q.new_empty((B, H, Sq), dtype=torch.float32)
    elif lse.shape != (B, H, Sq) or lse.dtype != torch.float32 or lse.stride(-1) != 1 or lse.device != device:
        raise ValueError(f"lse must be an fp32 (B, H, Sq) tensor on {device} with a contiguous last dim")
    args = (
        _ext.ABI_VERSION, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), B, H, Sq, Sk, D,
        *_strides3(q), *_strides3(k), *_strides3(v), *_strides3(out), *lse.stride()[:2], scale,
        block_index.data_ptr(), *block_index.stride()[:3], *counts, block_index.shape[3],
    )
    rc = _ext.attn_sparse(device, *args, 0, _ext.H3A_WORKSPACE_ASK)
    if rc == _ext.H3A_NEED_WORKSPACE:
        need = _ext.attn_sparse_workspace_size(device, *args, 0, 0)
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        rc = _ext.attn_sparse(device, *args, workspace.data_ptr(), need)
    if rc != _ext.H3A_OK:
        _ext.check(_ext.load_library(), rc)
    return out, lse


class BlockSparseKernel:
    """Block-sparse attention with the call form of :func:`flash_attn_func`: each
    query block attends to a share ``keep`` of the key blocks (rounded up, one at
    least), the marked ones of ``always`` first."""

    def __init__(self, keep: float, *, always: torch.Tensor | None = None) -> None:
        if not 0.0 < keep <= 1.0:
            raise ValueError(f"keep must be in (0, 1], got {keep}")
        self.keep, self.always = float(keep), always

    def __call__(
        self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float | None = None, causal: bool = False
    ) -> tuple[torch.Tensor, torch.Tensor]:
        if causal:
            raise RuntimeError("H3 sparse HIP attention supports only non-causal attention")
        # (Less 1e-9: the product may pass the whole number that is meant, as 0.07 *
        # 100 does 7.)
        topk = max(1, math.ceil((self.keep - 1e-9) * _blocks(k.shape[1], BLOCK_K)))
        return sparse_attn_func(q, k, v, select_key_blocks(q, k, topk, always=self.always), softmax_scale=softmax_scale)
