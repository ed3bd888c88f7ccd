"""BlockSparseKernel keeps the documented share of the key blocks, rounded up,
whatever the share's binary form."""

from __future__ import annotations

import pytest
import torch

from h3_flash_amd import BlockSparseKernel, sparse_attention


@pytest.mark.parametrize(
    "keep, blocks, topk",
    [
        (0.07, 100, 7),  # 0.07 * 100 = 7.000000000000001
        (0.55, 100, 55),
        (0.14, 50, 7),
        (0.07, 99, 7),
        (0.07, 101, 8),
        (5 / 6, 6, 5),
        (1 / 3, 3, 1),
        (2 / 3, 7168, 4779),
        (0.2, 780, 156),
        (1.0, 780, 780),
        (1e-12, 5, 1),
        (0.999, 7168, 7161),
    ],
)
def test_share_of_the_key_blocks(monkeypatch, keep, blocks, topk):
    seen = []
    monkeypatch.setattr(sparse_attention, "select_key_blocks", lambda q, k, n, always=None: seen.append(n))
    monkeypatch.setattr(sparse_attention, "sparse_attn_func", lambda *args, **kwargs: None)
    k = torch.empty((1, 64 * blocks - 63, 1, 128), dtype=torch.bfloat16)
    BlockSparseKernel(keep)(k, k, k)
    assert seen == [topk]
