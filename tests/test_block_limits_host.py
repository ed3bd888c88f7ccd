"""Limits of the block operators that the host decides: launches of few tokens
past 2^32 work items."""

from __future__ import annotations

import ctypes

import pytest

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
