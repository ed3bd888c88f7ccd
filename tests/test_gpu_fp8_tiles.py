"""Every tile form of the 8-bit product against 64 bits: each shape, plain and gated,
with either result, its reduction whole, in pieces, in pieces behind rounds of whole
tiles, and longer than the scales that a tile holds at once."""

from __future__ import annotations

import ctypes

import pytest
import torch

from h3_flash_amd import _ext, fused_linear_fp8
from test_gpu_fp8 import BF16, DEV, E8M0, F32, _check, _operands, _randn

pytestmark = pytest.mark.gpu

# m, k, n, gated, 8-bit result
CASES = [
    # 128 features x 32, 64, 96 and 128 tokens
    (33, 48, 16, False, False), (33, 48, 16, False, True), (33, 48, 24, True, False), (33, 17600, 16, False, True), (40, 17600, 136, True, False),
    (97, 2064, 8208, False, False), (97, 2064, 8208, False, True), (97, 2064, 4112, True, False), (33, 20800, 24, False, False),
    (33, 20800, 16, True, False), (33, 4112, 16400, True, False), (1600, 17600, 528, False, True), (33, 17600, 8208, True, False),
    (1000, 144, 1048, False, False), (1000, 144, 1040, False, True), (1000, 144, 536, True, False), (33, 4112, 24, False, False),
    (33, 4112, 16, True, False), (257, 4112, 11200, False, False), (130, 4112, 8208, True, False), (1000, 17600, 2064, False, True),
    (520, 272, 2072, False, False), (520, 272, 2064, False, True), (520, 272, 1048, True, False),
    (1000, 48, 1048, False, False), (1000, 48, 1040, False, True), (1000, 48, 536, True, False), (97, 8208, 1048, False, False),
    (97, 8208, 528, True, False), (800, 8208, 4800, False, False), (1000, 8208, 2064, True, False), (700, 17600, 4112, False, True),
    # 256 features x 128, 192 and 256 tokens
    (800, 48, 4808, False, False), (800, 48, 4800, False, True), (130, 48, 8208, True, False), (33, 48, 16, True, True), (33, 17600, 16, True, True),
    (700, 14400, 2064, False, False), (300, 14400, 4112, False, False), (1000, 11200, 4800, False, False), (390, 11200, 4800, True, False), (300, 14400, 2072, True, False), (200, 4112, 16400, True, False), (1000, 17600, 4112, False, True),
    (1300, 48, 6400, False, False), (1300, 48, 6400, False, True), (130, 48, 16408, True, False), (130, 48, 16400, True, True),
    (130, 14400, 8208, False, False), (130, 14400, 4112, True, False), (1300, 8208, 11200, False, False), (257, 4112, 16400, True, False),
    (520, 17600, 8208, True, False), (130, 17600, 16400, True, True),
    (1000, 48, 11208, False, False), (1000, 48, 11200, False, True), (200, 48, 16400, True, False), (200, 48, 16400, True, True),
    (1000, 11200, 4112, False, False), (1000, 11200, 2064, True, False), (1000, 4112, 16400, False, False), (390, 4112, 16400, True, False),
    (1600, 17600, 4112, True, False), (1000, 17600, 11200, False, True), (200, 17600, 16400, True, True),
]


@pytest.mark.parametrize("m, k, n, gated, quantize", CASES)
def test_tiles(m, k, n, gated, quantize):
    i = CASES.index((m, k, n, gated, quantize))
    a, a_scale, w, w_scale = _operands(m, k, n, "fp8", gated)
    rows = 2 * n if gated else n
    # the epilogue's parts in turn: none, a bias, all of them, a residual
    b = _randn(rows, seed=1, scale=0.3, dtype=(BF16, F32)[i % 2]) if i % 4 in (1, 2) else None
    r = _randn(m, n, seed=2, scale=2.0) if i % 4 > 1 else None
    g = _randn(7, n, seed=3, dtype=(F32, BF16)[i % 2]) if i % 4 == 2 else None
    index = None if g is None else torch.arange(m, device=DEV, dtype=(torch.int32, torch.int64)[i % 2]) * 7 // m
    rest = dict(activation=(None, "silu", "gelu", "gelu_tanh", "relu")[i % 5], gated=gated, residual=r, gate=g, index=index)
    got = fused_linear_fp8(a, w, w_scale, b, x_scale=a_scale, quantize=quantize, **rest)
    _check(got, quantize, a, a_scale, w, w_scale, b, **rest)


def test_rows_after_the_last_are_left_as_they_were():
    # tiles that reach past m, into a buffer with room behind it
    for m in (33, 100, 300, 1000):
        a, a_scale, w, w_scale = _operands(m, 272, 2056, "fp8", False)
        out = torch.full((m + 300, 2056), 3.0, dtype=BF16, device=DEV)
        fused_linear_fp8(a, w, w_scale, x_scale=a_scale, out=out[:m])
        assert torch.equal(out[:m], fused_linear_fp8(a, w, w_scale, x_scale=a_scale)) and (out[m:] == 3).all()


# (a last tile of one row, of most rows; 256 x 256, 192 and 128 and 128 x 32 tiles)
@pytest.mark.parametrize("m, k, n, gated", [(1025, 48, 11200, False), (1000, 48, 11200, False), (1345, 48, 6400, False), (257, 48, 16400, True),
                                            (33, 48, 16, False), (130, 48, 16400, True)])
@pytest.mark.parametrize("y8", [False, True])
def test_nothing_behind_a_result_is_written(m, k, n, gated, y8):
    a, a_scale, w, w_scale = _operands(m, k, n, "fp8", gated)
    a_scale, w_scale = (torch.nn.functional.pad(s.view(torch.uint8), (0, 16 - s.shape[1])) for s in (a_scale, w_scale))
    pitch = (n + 127) // 128 // 16 * 16 + 16
    y = torch.full((m + 300, n if y8 else 2 * n), 91, dtype=torch.uint8, device=DEV)
    ys = torch.full((m + 300, pitch), 92, dtype=torch.uint8, device=DEV)
    residual = _randn(m, n, seed=2)
    args = _ext.LinearFp8Args(
        abi_version=_ext.ABI_VERSION, x=a.data_ptr(), x_dtype=4, x_scale=a_scale.data_ptr(), weight=w.data_ptr(), weight_scale=w_scale.data_ptr(),
        residual=residual.data_ptr(), y=y.data_ptr(), y_dtype=4 if y8 else 0, y_scale=ys.data_ptr() if y8 else 0, m=m, k=k, n=n, x_stride=k,
        x_scale_stride=16, weight_stride=k, weight_scale_stride=16, residual_stride=n, y_stride=n, y_scale_stride=pitch, gated=int(gated))
    assert _ext.load_library().h3a_linear_fp8(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == _ext.H3A_OK
    groups = (n + 127) // 128
    assert (y[m:] == 91).all() and (ys[m:] == 92).all() and (ys[:, groups:] == 92).all() and (y8 or (ys == 92).all())
    want = fused_linear_fp8(a, w, w_scale[:, :1].view(E8M0), x_scale=a_scale[:, :1].view(E8M0), gated=gated, residual=residual, quantize=y8)
    want, scale = want if y8 else (want, None)
    assert torch.equal(y[:m], want.view(torch.uint8)) and (not y8 or torch.equal(ys[:m, :groups], scale.view(torch.uint8)))


@pytest.mark.parametrize("m", [300, 1500])
def test_scales_that_differ_from_block_to_block(m):
    # a scale read for the wrong token, feature block or K block shows: each is a
    # power of two of its own, the values are ones
    k, n = 128 * 21, 2 * 272
    one = torch.ones((m, k), device=DEV).to(torch.float8_e4m3fn)
    w = torch.ones((n, k), device=DEV).to(torch.float8_e4m3fn)
    i, j = torch.arange(m, device=DEV)[:, None], torch.arange(21, device=DEV)
    xe, we = (i * 7 + j * 3) % 5, (torch.arange(6, device=DEV)[:, None] * 5 + j * 2) % 7
    xs, ws = ((127 + e).to(torch.uint8).view(torch.float8_e8m0fnu) for e in (xe, we))
    for gated in (False, True):
        got = fused_linear_fp8(one, w, ws if gated else ws[:5], x_scale=xs, gated=gated)
        z = 128 * (2.0 ** xe.double()) @ (2.0 ** we.double()).t()  # of each block of features
        if gated:  # 272 features: blocks 0 to 2 of the values, 3 to 5 of the gates
            want = (z[:, :3] * z[:, 3:]).repeat_interleave(128, 1)[:, :272]
        else:
            want = z[:, :5].repeat_interleave(128, 1)[:, :n]
        assert torch.equal(got, want.to(BF16))
