"""What the host refuses of the block operators' calls: launches of few tokens past
2^32 work items, results over their operands."""

from __future__ import annotations

import ctypes

import pytest
import torch

from h3_flash_amd import _ext

P = 0x100000  # never read: the calls below end before any launch


@pytest.fixture(scope="module")
def lib():
    return _ext.load_library()


def _linear(m, k, n, gated=0, **kw):
    base = dict(abi_version=_ext.ABI_VERSION, x=P, weight=2 * P, y=3 * P, m=m, k=k, n=n, x_stride=k, weight_stride=k, y_stride=n,
                gated=gated)
    return _ext.LinearArgs(**{**base, **kw})


@pytest.mark.parametrize("m", [1, 16, 17, 32])
@pytest.mark.parametrize(
    "gated, n, fits",
    [
        # 256 work items take 64 rows of the weight at this width: 2^32 from 2^30 rows on
        (1, 2**29 - 32, True),
        (1, 2**29 - 24, False),
        (1, 2**29 + 8, False),
        (1, 2**30 - 8, False),
        (0, 2**30 - 64, True),
        (0, 2**30 - 56, False),
        (0, 2**30 - 8, False),
    ],
)
def test_few_tokens_past_the_work_items_of_a_launch_are_refused(lib, m, gated, n, fits):
    # (the query plans the launch as the call does, and launches nothing)
    rc = lib.h3a_linear_workspace_size(ctypes.byref(_linear(m, 8, n, gated)))
    if fits:
        assert rc == 0, _ext.last_error(lib)
    else:
        assert rc == _ext.H3A_EUNSUPPORTED and "grid too large" in _ext.last_error(lib)


# The result apart from the operands: 8 tokens of 64 columns, 32 features.
A = 0x1000000
APART = dict(x=A, weight=A + 0x10000, y=A + 0x20000)


@pytest.mark.skipif(torch.cuda.is_available(), reason="fake device pointers: GPU-less hosts only")
@pytest.mark.parametrize(
    "overlaps, kw",
    [
        (True, dict(y=A)),  # x itself
        (True, dict(y=A + 7 * 128 + 112)),  # its last row's last columns
        (True, dict(y=A + 0x10000)),  # the weight
        (True, dict(y=A + 0x10000 - 8 * 64 + 16)),  # the result's last row ends in it
        (False, dict(y=A + 8 * 128)),  # right behind x
        (False, dict(y=A + 0x10000 - 8 * 64)),  # right before the weight
        # columns of one buffer: apart, one chunk too far, wrapped into x's next row
        (False, dict(x_stride=96, y_stride=96, y=A + 128)),
        (True, dict(x_stride=96, y_stride=96, y=A + 112)),
        (True, dict(x_stride=88, y_stride=88, y=A + 128)),
        # the residual itself, at the same pitch or in one row; any other overlap with it
        (False, dict(residual=A + 0x20000, residual_stride=32)),
        (False, dict(residual=A + 0x20000, residual_stride=64, m=1)),
        (True, dict(residual=A + 0x20000, residual_stride=64)),
        (True, dict(residual=A + 0x20000 + 64, residual_stride=32)),
        (False, dict(residual=A + 0x20000 + 64, residual_stride=64, y_stride=64)),
        (True, dict(bias=A + 0x20000 + 16)),
        (False, dict(bias=A + 0x20000 + 64, y_stride=64)),  # beside the result's rows
        (True, dict(gate=A + 0x20000 + 7 * 64, gate_stride=32, table_rows=3, index=P, index_dtype=3, n_index=1)),
        (True, dict(gate=A + 0x20000 - 128, gate_stride=32, table_rows=3, index=P, index_dtype=3, n_index=1)),
    ],
)
def test_a_result_that_overlaps_an_operand_is_refused(lib, overlaps, kw):
    rc = lib.h3a_linear(ctypes.byref(_linear(**{**dict(m=8, k=64, n=32), **APART, **kw})), None)
    # (without a device the accepted ones end in a failed launch)
    assert rc == (_ext.H3A_EINVAL if overlaps else _ext.H3A_ELAUNCH), _ext.last_error(lib)
    assert ("overlap" in _ext.last_error(lib)) == overlaps
