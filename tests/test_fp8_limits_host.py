"""The largest launches of the 8-bit layers' roundings: what needs more than 2^32 - 1 work
items in workgroups of 256 is refused before it, one group of rows less is not. (Pointers
are made up and the host has no device, where what is not refused ends as a failed launch.)"""

from __future__ import annotations

import ctypes

import pytest
import torch

from h3_flash_amd import _ext

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="fake device pointers: GPU-less hosts only")
X, Q, SCALE, W = 1 << 40, 1 << 42, 1 << 44, 1 << 39
MOST_ROWS = 64 * (2**24 - 1)  # groups of rows: 64 a workgroup
MOST_BLOCKS = 2**24 - 1
UNSUPPORTED, ELAUNCH = _ext.H3A_EUNSUPPORTED, _ext.H3A_ELAUNCH


@pytest.fixture(scope="module")
def lib():
    return _ext.load_library()


def _quantize(rows, cols=16, **kw):
    scale_stride = (cols + 127) // 128 // 16 * 16 + 16
    return _ext.QuantizeFp8Args(**{**dict(abi_version=_ext.ABI_VERSION, x=X, x_dtype=0, q=Q, scale=SCALE, rows=rows, cols=cols, block_rows=1,
                                          parts=1, x_stride=cols, q_stride=cols, scale_stride=scale_stride), **kw})


def _linear(m, k=16):
    return _ext.LinearFp8Args(abi_version=_ext.ABI_VERSION, x=X, x_dtype=0, weight=W, weight_scale=W + (1 << 30), y=SCALE, y_dtype=0, m=m, k=k,
                              n=8, x_stride=k, weight_stride=k, weight_scale_stride=16, y_stride=8)


@pytest.mark.parametrize("x_dtype", [_ext.H3A_DTYPE_BF16, _ext.H3A_DTYPE_F32])
@pytest.mark.parametrize("rows, cols", [(MOST_ROWS, 16), (MOST_ROWS, 128), (MOST_ROWS // 2, 144), (MOST_ROWS // 3, 384)])
def test_rows(lib, rows, cols, x_dtype):
    groups = (cols + 127) // 128
    assert rows * groups == MOST_ROWS
    assert lib.h3a_quantize_fp8(ctypes.byref(_quantize(rows, cols, x_dtype=x_dtype)), None) == ELAUNCH
    for more in (rows + 1, 2**30 // groups - 1, 2**30 // groups + 1):
        assert lib.h3a_quantize_fp8(ctypes.byref(_quantize(more, cols, x_dtype=x_dtype)), None) == UNSUPPORTED
        assert "too large" in _ext.last_error(lib)


def test_blocks(lib):
    # two blocks to every 128 rows
    for blocks, code in ((MOST_BLOCKS - 1, ELAUNCH), (MOST_BLOCKS + 1, UNSUPPORTED)):
        args = _quantize(64 * blocks, 256, block_rows=128)
        assert lib.h3a_quantize_fp8(ctypes.byref(args), None) == code, blocks


def test_bf16_rows_of_a_product(lib):
    assert lib.h3a_linear_fp8_required_workspace(ctypes.byref(_linear(MOST_ROWS))) > 0
    assert lib.h3a_linear_fp8_required_workspace(ctypes.byref(_linear(MOST_ROWS // 3, 272))) > 0
    for m, k in ((MOST_ROWS + 1, 16), (2**30 - 1, 16), (MOST_ROWS // 3 + 1, 272)):
        assert lib.h3a_linear_fp8_required_workspace(ctypes.byref(_linear(m, k))) == UNSUPPORTED, (m, k)
        assert "too large" in _ext.last_error(lib)
