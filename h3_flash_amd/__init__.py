"""MI355X-native attention hot path of H3-Flash (gfx950 HIP kernels).

The modules ``relayout``, ``fusions``, ``projection`` and
``context_parallel`` hold the rows around the attention call."""

from .attention import (
    DenseMiniMaxH3Processor,
    flash_attn_func,
    flash_attn_varlen_func,
    hip_forward_op,
    install_dense_hip,
    load_kernel,
    provenance,
)
from .context_parallel import chunked_attention, merge_attention
from .linear import fused_linear
from .prologue import fused_qk_norm_rope, fused_qknorm_rope
from .sparse_attention import BlockSparseKernel, select_key_blocks, sparse_attn_func

__all__ = [
    "BlockSparseKernel",
    "DenseMiniMaxH3Processor",
    "chunked_attention",
    "flash_attn_func",
    "flash_attn_varlen_func",
    "fused_linear",
    "fused_qk_norm_rope",
    "fused_qknorm_rope",
    "hip_forward_op",
    "install_dense_hip",
    "load_kernel",
    "merge_attention",
    "provenance",
    "select_key_blocks",
    "sparse_attn_func",
]
