"""GPU parity of the forms that the block operators take for long lists, extreme
scores, far-apart rows and long sequences, with the form pinned: a launch of
attention over lists that asks for a workspace runs its tiles in pieces with one
and whole without one (never as units of 32 rows), so both are compared here
whatever the rule that chooses between them."""

from __future__ import annotations

import math

import pytest
import torch

from h3_flash_amd import _ext, fused_linear, select_key_blocks, sparse_attn_func
from h3_flash_amd.fusions import fused_rmsnorm_residual_gate_rmsnorm_modulate
from oracle.block import linear_reference, sandwich_reference, select_reference, sparse_reference

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32 = torch.bfloat16, torch.float32


def _randn(*shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


def _within(got, want, bound, tag):
    some = ~want.isinf()
    assert torch.equal(got.isinf().cpu(), ~some.cpu()), (tag, "infinite")
    off = (got.double().to(want.device).reshape(want.shape) - want).abs() / bound.clamp_min(1e-37)
    worst = off[some].nan_to_num(nan=math.inf).max().item() if some.any() else 0.0
    assert worst <= 1.0, (tag, worst)


def _check(got, q, k, v, index, count=None, scale=None, tag=""):
    """Against 64 bits, elementwise, within the bound of the arithmetic."""

    c = lambda t: None if t is None else t.cpu()  # noqa: E731
    o, o_bound, l, l_bound = sparse_reference(c(q), c(k), c(v), c(index), c(count), scale)
    _within(got[0].cpu(), o, o_bound, (tag, "out"))
    _within(got[1].cpu(), l, l_bound, (tag, "lse"))


def _in_pieces_and_whole(q, k, v, index, count=None, scale=None):
    """The call's results in pieces and with every list whole."""

    B, Sq, H, D = q.shape
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty((B, H, Sq), device=DEV)
    counts = (0, 0, 0, 0) if count is None else (count.data_ptr(), *count.stride())
    args = (
        _ext.ABI_VERSION, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), B, H, Sq, k.shape[1], D,
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *lse.stride()[:2],
        1.0 / math.sqrt(D) if scale is None else scale,
        index.data_ptr(), *index.stride()[:3], *counts, index.shape[3],
    )
    assert _ext.attn_sparse_workspace_size(DEV, *args, 0, 0) > 0, "the launch was to run in pieces"
    pieces = sparse_attn_func(q, k, v, index, count, scale)
    assert _ext.attn_sparse(DEV, *args, 0, 0) == _ext.H3A_OK
    return (("pieces", pieces), ("whole", (out, lse)))


def _tall_keys(k, index, blocks, factor):
    """Scales the keys of the listed blocks at the given places of a list."""

    for at in blocks:
        n = int(index[at])
        k[0, 64 * n : 64 * (n + 1)] *= factor


# ---------------------------------------------------------------- attention in tiles


@pytest.mark.parametrize("Sq, H", [(257, 1), (300, 2)])
@pytest.mark.parametrize("factor", [12.0, 40.0, 300.0])
def test_extreme_scores_in_tiles(Sq, H, factor):
    # In every piece (an eighth of the list) the scores of its fifth block are far
    # above its first one's: by some 40 log2 units (the offset rises by powers of
    # two), 150 and 1,000 (the block's softmax is done again against its exact
    # max, from K in global memory). The last entry, the ragged block, as well.
    Sk, n = 64 * 63 - 27, 63
    q, k, v = (_randn(1, s, H, 128, seed=40 + i) for i, s in enumerate((Sq, Sk, Sk)))
    order = torch.randperm(n - 1, generator=torch.Generator().manual_seed(41)).tolist() + [n - 1]
    _tall_keys(k, order, [*range(4, n - 1, 8), n - 1], factor)
    index = torch.tensor(order, dtype=torch.int32, device=DEV).expand(1, H, -(-Sq // 256), n)
    for form, got in _in_pieces_and_whole(q, k, v, index):
        _check(got, q, k, v, index, tag=form)
    back = index.flip(-1).contiguous()  # the tall blocks before the others, too
    for form, got in _in_pieces_and_whole(q, k, v, back, scale=0.25):
        _check(got, q, k, v, back, scale=0.25, tag=(form, "reversed"))


def test_extreme_scores_in_many_whole_tiles():
    # More tiles than CUs: whole by themselves, an odd list.
    Sq, Sk, H, n = 5000, 1100, 20, 7
    q, k, v = (_randn(1, s, H, 128, seed=45 + i) for i, s in enumerate((Sq, Sk, Sk)))
    order = [3, 0, 11, 17, 8, 2, 14]
    _tall_keys(k, order, [3], 40.0)  # the ragged block
    _tall_keys(k, order, [5], 300.0)
    index = torch.tensor(order, dtype=torch.int32, device=DEV).expand(1, H, 20, n)
    out, lse = sparse_attn_func(q, k, v, index)
    for h in (0, 19):
        hs = slice(h, h + 1)
        _check((out[:, :, hs], lse[:, hs]), q[:, :, hs], k[:, :, hs], v[:, :, hs], index[:, hs], tag=h)


def test_rows_past_four_gib_in_tiles():
    # K and V rows 2.4 MB apart: the byte offsets of most blocks pass 32 bits
    S, stride, n = 2000, 1_200_000, 63
    base = torch.zeros(S * stride, dtype=BF16, device=DEV)
    k, v = (base.as_strided((1, S, 1, 128), (S * stride, stride, 128, 1), 256 * i) for i in range(2))
    k.copy_(_randn(1, S, 1, 128, seed=60))
    v.copy_(_randn(1, S, 1, 128, seed=61))
    k[0, 64 * 29 : 64 * 30] *= 40.0  # the second pass over K of a block past 4 GiB
    q = _randn(1, 300, 1, 128, seed=62)
    g = torch.Generator().manual_seed(63)
    index = torch.randint(0, 32, (1, 1, 2, n), generator=g, dtype=torch.int32)
    index[..., 45], index[..., 20] = 29, 31
    index = index.to(DEV)
    for form, got in _in_pieces_and_whole(q, k, v, index):
        _check(got, q, k.contiguous(), v.contiguous(), index, tag=form)


def test_entries_of_any_kind_in_tiles():
    # Valid entries between ones that name nothing, some twice, the ragged block
    # in the middle; counts that leave some pieces, or all, without a block.
    H, Sq, Sk, n = 3, 600, 64 * 30 - 5, 63
    q, k, v = (_randn(1, s, H, 128, seed=70 + i) for i, s in enumerate((Sq, Sk, Sk)))
    g = torch.Generator().manual_seed(71)
    index = torch.randint(-12, 42, (1, H, 3, n), generator=g, dtype=torch.int32)
    index[0, 0, 0, 30], index[0, 1, 1, 5:9] = 29, torch.tensor([1 << 30, -(1 << 31), 29, 29], dtype=torch.int32)
    index = index.to(DEV)
    count = torch.tensor([[[63, 3, 0], [9, 40, -4], [1, 99, 8]]], dtype=torch.int32, device=DEV)
    for form, got in _in_pieces_and_whole(q, k, v, index):
        _check(got, q, k, v, index, tag=form)
    for form, got in _in_pieces_and_whole(q, k, v, index, count):
        _check(got, q, k, v, index, count.clamp(0, n), tag=(form, "counts"))
        assert (got[0][:, 512:, 0] == 0).all() and torch.isneginf(got[1][:, 0, 512:]).all()


def test_results_do_not_vary_between_calls_in_any_form():
    for Sq, Sk, H, n in ((16, 3000, 4, 24), (257, 4000, 2, 63), (5000, 1100, 20, 7)):  # units, pieces, whole tiles
        q, k, v = (_randn(1, s, H, 128, seed=75 + i) for i, s in enumerate((Sq, Sk, Sk)))
        g = torch.Generator().manual_seed(78)
        index = torch.randint(0, -(-Sk // 64), (1, H, -(-Sq // 256), n), generator=g, dtype=torch.int32).to(DEV)
        first = sparse_attn_func(q, k, v, index)
        for _ in range(4):
            again = sparse_attn_func(q, k, v, index)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1]), (Sq, H, n)


# ---------------------------------------------------------------- long sequences


@pytest.mark.parametrize("H, S, n", [(40, 49920, 156), (2, 129024, 200)])
def test_long_sequences(H, S, n):
    # one GPU's whole block, and the longest sequence: three query blocks of the
    # first, a middle and the last head each
    q, k, v = (_randn(1, S, H, 128, seed=80 + i) for i in range(3))
    nq, nk = -(-S // 256), -(-S // 64)
    index = torch.rand((1, H, nq, nk), device=DEV, generator=torch.Generator(device=DEV).manual_seed(83)).topk(n, -1).indices.to(torch.int32)
    out, lse = sparse_attn_func(q, k, v, index)
    for h in {0, H // 2, H - 1}:
        hs = slice(h, h + 1)
        for i in (0, nq // 2, nq - 1):
            rows = slice(256 * i, min(256 * (i + 1), S))
            _check((out[:, rows, hs], lse[:, hs, rows]), q[:, rows, hs], k[:, :, hs], v[:, :, hs], index[:, hs, i : i + 1], tag=(h, i))


def test_selection_over_the_longest_sequence():
    S = 129024 - 100
    q, k = _randn(1, S, 1, 128, seed=90), _randn(1, S, 1, 128, seed=91)
    assert torch.equal(select_key_blocks(q, k, 403).cpu(), select_reference(q.cpu(), k.cpu(), 403))


@pytest.mark.parametrize(
    "m, k, n, activation, gated, bias, residual, gate",
    [
        (8200, 136, 520, "silu", True, BF16, True, F32),
        (16384, 72, 264, "gelu", False, F32, True, BF16),
        (16641, 136, 1032, None, False, BF16, True, BF16),
        (16641, 72, 520, "silu", True, None, False, None),
        (49920, 264, 1544, "gelu_tanh", False, BF16, True, F32),
        (129024, 72, 264, "relu", False, F32, False, None),
    ],
)
def test_linear_over_long_sequences(m, k, n, activation, gated, bias, residual, gate):
    rows = 2 * n if gated else n
    x, w = _randn(m, k, seed=m), _randn(rows, k, seed=k, scale=k**-0.5)
    b = None if bias is None else _randn(rows, seed=1, scale=0.3, dtype=bias)
    r = _randn(m, n, seed=2, scale=2.0) if residual else None
    g = None if gate is None else _randn(9, n, seed=3, dtype=gate)
    index = None if gate is None else torch.arange(m, device=DEV) * 9 // m
    got = fused_linear(x, w, b, activation=activation, gated=gated, residual=r, gate=g, index=index)
    _within(got, *linear_reference(x, w, b, activation, gated, r, g, index), (m, k, n))


@pytest.mark.parametrize("rows, cols, tables", [(49920, 5376, BF16), (20000, 1001, BF16), (17000, 5120, F32), (49920, 1024, F32)])
def test_norms_over_long_sequences(rows, cols, tables):
    r, b = _randn(rows, cols, seed=100, scale=2.0), _randn(rows, cols, seed=101)
    bw, w = (1 + _randn(cols, seed=102 + i, scale=0.1, dtype=F32) for i in range(2))
    gate, scale, shift = (_randn(9, cols, seed=104 + i, scale=0.3, dtype=tables) for i in range(3))
    index = torch.arange(rows, device=DEV) * 9 // rows
    hidden, normed = fused_rmsnorm_residual_gate_rmsnorm_modulate(r, b, bw, gate, w, scale, shift, index, 1e-5, residual_scale=0.75)
    for part in (slice(0, 700), slice(rows // 2 - 3, rows // 2 + 500), slice(rows - 333, rows)):
        h, hb, n, nb = sandwich_reference(r[part], b[part], bw, gate, w, scale, shift, index[part], 1e-5, 0.75)
        _within(hidden[part], h, hb, (rows, cols, "hidden"))
        _within(normed[part], n, nb, (rows, cols, "normed"))
