"""GPU parity of key-block selection (equal indices) and of attention over block
lists (elementwise within the bound of its arithmetic, oracle.block)."""

from __future__ import annotations

import math

import pytest
import torch

from h3_flash_amd import BlockSparseKernel, flash_attn_func, select_key_blocks, sparse_attn_func
from oracle.block import select_reference, sparse_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16 = torch.bfloat16


def _randn(*shape, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(BF16)


def _lists(B, H, nq, nk, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand((B, H, nq, nk), generator=g).topk(min(n, nk), -1).indices.to(torch.int32).to(DEV)


def _check(got, want, tag=""):
    out, lse = got
    o, o_bound, l, l_bound = want
    assert out.dtype == BF16 and lse.dtype == torch.float32
    worst = ((out.double().cpu() - o).abs() / o_bound.clamp_min(1e-37)).nan_to_num(nan=math.inf).max().item()
    assert worst <= 1.0, (tag, "out", worst)
    lse = lse.double().cpu()
    assert torch.equal(lse.isinf(), l.isinf()), (tag, "rows without keys")
    some = ~l.isinf()
    if some.any():
        worst = ((lse - l).abs() / l_bound.clamp_min(1e-30))[some].nan_to_num(nan=math.inf).max().item()
        assert worst <= 1.0, (tag, "lse", worst)


def _parity(q, k, v, index, count=None, scale=None, tag="", **kwargs):
    got = sparse_attn_func(q, k, v, index, count, scale, **kwargs)
    _check(got, sparse_reference(q.cpu(), k.cpu(), v.cpu(), index.cpu(), None if count is None else count.cpu(), scale), tag)
    return got


# ---------------------------------------------------------------- selection


@pytest.mark.parametrize(
    "B, Sq, Sk, H, topk",
    [
        (1, 1, 1, 1, 1),
        (2, 257, 65, 3, 1),
        (1, 700, 1001, 2, 5),
        (1, 1560, 1560, 5, 7),
        (1, 300, 4096, 1, 64),
        (1, 256, 4097, 2, 65),  # more than one key a lane, all of them
        (1, 33, 16385, 1, 100),
        (1, 20, 66000, 1, 300),
        (1, 3, 263000, 1, 1000),  # a workgroup per row
        (1, 5, 64, 2, 9),  # topk past the blocks there are
    ],
)
def test_select_parity(B, Sq, Sk, H, topk):
    q, k = _randn(B, Sq, H, 128, seed=Sq), _randn(B, Sk, H, 128, seed=Sk)
    got = select_key_blocks(q, k, topk)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), select_reference(q.cpu(), k.cpu(), topk))


def test_select_marked_blocks_come_first():
    q, k = _randn(1, 300, 2, 128, seed=1), _randn(1, 1300, 2, 128, seed=2)
    always = torch.zeros(21, dtype=torch.bool)
    always[[0, 3, 20]] = True
    for topk in (1, 2, 3, 4, 9):
        got = select_key_blocks(q, k, topk, always=always.to(DEV))
        assert torch.equal(got.cpu(), select_reference(q.cpu(), k.cpu(), topk, always)), topk
    assert torch.equal(select_key_blocks(q, k, 4, always=always), select_key_blocks(q, k, 4, always=always.to(DEV).int()))


def test_select_ties_go_to_the_lowest_index():
    # equal key blocks: every score of a row the same, but for two
    q = _randn(1, 256, 1, 128, seed=3)
    k = _randn(1, 64, 1, 128, seed=4).repeat(1, 200, 1, 1)
    assert torch.equal(select_key_blocks(q, k, 11).cpu().flatten(), torch.arange(11, dtype=torch.int32))
    top = q.float().mean(1, keepdim=True).to(BF16)
    k[:, 64 * 77 : 64 * 78], k[:, 64 * 150 : 64 * 151] = 8 * top, 8 * top
    want = torch.tensor([*range(9), 77, 150], dtype=torch.int32)
    assert torch.equal(select_key_blocks(q, k, 11).cpu().flatten(), want)
    # zeros of either sign are one score
    k = torch.zeros_like(k)
    k[:, 64 * 5 :] *= -1.0
    assert torch.equal(select_key_blocks(q, k, 6).cpu().flatten(), torch.arange(6, dtype=torch.int32))


def test_select_values_that_are_not_finite():
    q, k = _randn(1, 256, 1, 128, seed=5).abs(), _randn(1, 640, 1, 128, seed=6)
    k[0, 70, 0, 3] = float("nan")  # block 1: NaN
    k[0, 200] = -float("inf")  # block 3: -inf
    k[0, 400] = float("inf")  # block 6: +inf
    assert torch.equal(select_key_blocks(q, k, 9).cpu(), select_reference(q.cpu(), k.cpu(), 9))
    assert 6 in select_key_blocks(q, k, 1).flatten().tolist()
    assert select_key_blocks(q, k, 9).flatten().tolist() == [0, 1, 2, 4, 5, 6, 7, 8, 9]  # NaN is -inf, and comes first


def test_select_strided_views():
    qkv = _randn(2, 600, 3 * 4, 128, seed=7)
    q, k, _ = qkv.chunk(3, dim=2)
    assert torch.equal(select_key_blocks(q, k, 4).cpu(), select_reference(q.cpu(), k.cpu(), 4))
    bhsd = _randn(2, 3, 600, 128, seed=8).transpose(1, 2)
    assert torch.equal(select_key_blocks(bhsd, bhsd, 3).cpu(), select_reference(bhsd.cpu(), bhsd.cpu(), 3))


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize(
    "B, Sq, Sk, H, n",
    [
        (1, 1, 1, 1, 1),
        (1, 1, 700, 3, 4),
        (2, 33, 65, 2, 2),  # the last block holds one key
        (1, 16, 12480, 8, 24),
        (1, 300, 1001, 2, 3),
        (1, 257, 4000, 1, 63),  # longer lists than units take
        (1, 513, 2000, 2, 1),
        (1, 1560, 1560, 4, 9),
        (1, 4095, 4095, 2, 16),
        (2, 2049, 640, 3, 10),
        (1, 520, 20000, 1, 200),
    ],
)
def test_attention_parity(B, Sq, Sk, H, n):
    q, k, v = (_randn(B, s, H, 128, seed=i + Sq) for i, s in enumerate((Sq, Sk, Sk)))
    index = _lists(B, H, -(-Sq // 256), -(-Sk // 64), n, seed=Sk)
    _parity(q, k, v, index)


@pytest.mark.parametrize("Sq, H", [(40, 2), (700, 2), (5000, 20)])
def test_counts_and_rows_without_keys(Sq, H):
    Sk, nq = 1100, -(-Sq // 256)
    q, k, v = (_randn(1, s, H, 128, seed=i) for i, s in enumerate((Sq, Sk, Sk)))
    index = _lists(1, H, nq, 18, 7, seed=9)
    g = torch.Generator().manual_seed(10)
    count = torch.randint(-1, 10, (1, H, nq), generator=g, dtype=torch.int32).to(DEV)
    count[0, 0, 0], count[0, -1, -1] = 0, 12
    got = sparse_attn_func(q, k, v, index, count)
    clamped = count.clamp(0, 7)
    # every row against the reference on a few heads
    for h in ([0, H - 1] if H > 2 else range(H)):
        hs = slice(h, h + 1)
        want = sparse_reference(q[:, :, hs].cpu(), k[:, :, hs].cpu(), v[:, :, hs].cpu(), index[:, hs].cpu(), clamped[:, hs].cpu())
        _check((got[0][:, :, hs], got[1][:, hs]), want, h)
    assert (got[0][:, : min(Sq, 256), 0] == 0).all() and got[1][:, 0, : min(Sq, 256)].isinf().all()


@pytest.mark.parametrize("Sq", [20, 300, 3000])
def test_entries_in_any_order_twice_and_outside(Sq):
    H, Sk, nq = 2, 777, -(-Sq // 256)
    q, k, v = (_randn(1, s, H, 128, seed=20 + i) for i, s in enumerate((Sq, Sk, Sk)))
    index = torch.tensor([12, -1, 3, 99, 3, 13, 0, 1 << 30, -(1 << 31), 12, 12], dtype=torch.int32, device=DEV).expand(1, H, nq, 11)
    _parity(q, k, v, index)  # 12 (the ragged block) three times, 3 twice
    assert torch.equal(sparse_attn_func(q, k, v, index)[0], sparse_attn_func(q, k, v, index.contiguous())[0])
    none = torch.full((1, H, nq, 70), -5, dtype=torch.int32, device=DEV)
    out, lse = sparse_attn_func(q, k, v, none)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_all_blocks_are_dense_attention():
    for Sq, Sk, H in ((50, 200, 2), (1000, 1000, 2), (4096, 4096, 4)):
        q, k, v = (_randn(1, s, H, 128, seed=30 + i) for i, s in enumerate((Sq, Sk, Sk)))
        nk = -(-Sk // 64)
        index = torch.arange(nk, dtype=torch.int32, device=DEV).expand(1, H, -(-Sq // 256), nk)
        out, lse = sparse_attn_func(q, k, v, index)
        ref, ref_lse = flash_attn_func(q, k, v)
        # two bf16 outputs of the same sums in another order, weights rounded to bf16
        assert (out.float() - ref.float()).abs().max() <= 2e-2 and (lse - ref_lse).abs().max() <= 1e-3


@pytest.mark.parametrize("Sq", [33, 600])
def test_extreme_scores(Sq):
    # scores far above the first block's, up to thousands of log2 units, in
    # either order of the list
    H, Sk = 1, 640
    q, k, v = (_randn(1, s, H, 128, seed=40 + i) for i, s in enumerate((Sq, Sk, Sk)))
    k[0, 64 * 4 : 64 * 5] *= 40.0
    k[0, 64 * 7 + 1] *= 300.0
    for order in ([0, 1, 4, 7], [7, 4, 1, 0], [4, 0, 2, 3, 9, 7, 8]):
        index = torch.tensor(order, dtype=torch.int32, device=DEV).expand(1, H, -(-Sq // 256), len(order))
        _parity(q, k, v, index, tag=order)
    _parity(q, k, v, index, scale=0.5, tag="scale")


def test_strided_views_and_given_outputs():
    H, S = 3, 900
    q, k, v = _randn(2, S, 3 * H, 128, seed=50).chunk(3, dim=2)
    index = _lists(2, H, 4, 15, 6, seed=51)
    wide = torch.zeros((2, H, 4, 12), dtype=torch.int32, device=DEV)
    wide[..., 3:9] = index
    out = torch.full((2, S + 3, H + 2, 128), 3.0, dtype=BF16, device=DEV)
    lse = torch.full((2, H + 1, S), 5.0, device=DEV)
    count = torch.full((4, H, 2), 6, dtype=torch.int32, device=DEV).permute(2, 1, 0)
    got = _parity(q, k, v, wide[..., 3:9], count, out=out[:, :S, :H], lse=lse[:, :H])
    assert got[0].data_ptr() == out.data_ptr()
    assert (out[:, S:] == 3.0).all() and (out[:, :, H:] == 3.0).all() and (lse[:, H:] == 5.0).all()


def test_views_past_four_gib():
    # K and V rows 2.4 MB apart: byte offsets beyond 32 bits, in tiles and units
    S, stride = 2000, 1_200_000
    base = torch.zeros(S * stride, dtype=BF16, device=DEV)
    k, v = (base.as_strided((1, S, 1, 128), (S * stride, stride, 128, 1), 256 * i) for i in range(2))
    k.copy_(_randn(1, S, 1, 128, seed=60))
    v.copy_(_randn(1, S, 1, 128, seed=61))
    for Sq in (16, 300):
        q = _randn(1, Sq, 1, 128, seed=62)
        _parity(q, k, v, _lists(1, 1, -(-Sq // 256), 32, 9, seed=63), tag=Sq)
    assert torch.equal(select_key_blocks(q, k, 5), select_key_blocks(q, k.contiguous(), 5))


def test_nothing_to_do():
    q, k = _randn(1, 300, 2, 128, seed=70), _randn(1, 100, 2, 128, seed=71)
    index = torch.zeros((1, 2, 2, 0), dtype=torch.int32, device=DEV)
    for kk, ii in ((k, index), (k[:, :0], index), (k[:, :0], torch.zeros((1, 2, 2, 3), dtype=torch.int32, device=DEV))):
        out, lse = sparse_attn_func(q, kk, kk, ii)
        assert (out == 0).all() and torch.isneginf(lse).all()
    assert sparse_attn_func(q[:, :0], k, k, torch.zeros((1, 2, 0, 3), dtype=torch.int32, device=DEV))[0].shape == (1, 0, 2, 128)
    assert select_key_blocks(q[:, :0], k, 2).shape == (1, 2, 0, 2)
    assert select_key_blocks(q, k[:, :0], 2).shape == (1, 2, 2, 0)


def test_the_longest_lists():
    n = 7168
    q, k, v = (_randn(1, s, 1, 128, seed=80 + i) for i, s in enumerate((3, 1024, 1024)))
    g = torch.Generator().manual_seed(81)
    index = torch.randint(-2, 18, (1, 1, 1, n), generator=g, dtype=torch.int32).to(DEV)
    _parity(q, k, v, index)
    with pytest.raises(RuntimeError, match="at most 7168"):
        sparse_attn_func(q, k, v, torch.zeros((1, 1, 1, n + 1), dtype=torch.int32, device=DEV))


def test_kernel_for_a_processor():
    q, k, v = (_randn(1, 1500, 2, 128, seed=90 + i) for i in range(3))
    out, lse = BlockSparseKernel(keep=0.25)(q, k, v, causal=False)
    index = select_key_blocks(q, k, 6)
    want = sparse_attn_func(q, k, v, index)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    with pytest.raises(RuntimeError):
        BlockSparseKernel(keep=0.25)(q, k, v, causal=True)
    with pytest.raises(ValueError):
        BlockSparseKernel(keep=0.0)


def test_refusals():
    q, k = _randn(1, 300, 2, 128, seed=91), _randn(1, 100, 2, 128, seed=92)
    index = torch.zeros((1, 2, 2, 1), dtype=torch.int32, device=DEV)
    count = torch.ones((1, 2, 2), dtype=torch.int32, device=DEV)
    for kind, args in (
        (TypeError, (q.float(), k, k, index)),
        (ValueError, (q[..., :64], k[..., :64], k[..., :64], index)),
        (RuntimeError, (q, k[:, :, :1], k[:, :, :1], index)),
        (ValueError, (q, k, k[:, :50], index)),
        (ValueError, (q, k, k, index[:, :, :1])),
        (ValueError, (q, k, k, index.long())),
        (ValueError, (q, k, k, index.cpu())),
        (ValueError, (q, k, k, index, count[:, :1])),
        (ValueError, (q, k, k, index, count.long())),
        (ValueError, (q, k, k, index, None, 0.0)),
    ):
        with pytest.raises(kind):
            sparse_attn_func(*args)
    for kind, args, kwargs in (
        (ValueError, (q, k, 0), {}),
        (ValueError, (q, k, 1), {"always": torch.ones(3, dtype=torch.bool)}),
        (RuntimeError, (q, k[:, :, :1], 1), {}),
        (TypeError, (q, k.float(), 1), {}),
    ):
        with pytest.raises(kind):
            select_key_blocks(*args, **kwargs)
