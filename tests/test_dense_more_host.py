"""Dense attention without a GPU, continued: the ends of its ranges, and what reaches the kernels."""
from __future__ import annotations

import ctypes

import pytest

from tasft_amd import _native

FAKE = ctypes.c_void_p(16)  # never dereferenced


@pytest.mark.parametrize(("scale", "cap"), [(1e-16, 1e30), (1e-30, 1e10), (1.0, 9e37)])
def test_quotients_that_fp32_does_not_hold(scale, cap):
    """scale / cap as 0 or with fewer bits: no scores could be made of it."""
    lib = _native.load_library()
    st, sl = _native.kept_strides((64 * 10 * 4, 640, 64, 1)), _native.kept_strides((40, 10, 1))
    rc = lib.tasft_dense_fwd(FAKE, FAKE, FAKE, FAKE, FAKE, None, None, None, None, None, 2, 10, 4, 2, 10, 64, st, st, st, st,
                             sl, scale, cap, 1, 0, None)
    assert rc == -1 and b"out of range" in lib.tasft_last_error()
    rc = lib.tasft_chunk_scored_fwd(
        FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, None, None, 0, None, 0, 2, 200, 4, 2, 100, 64, 64, 3, 8, 4,
        3, 1, st, st, st, st, st, 3, scale, cap, 1, 0, None)
    assert rc == -1 and b"out of range" in lib.tasft_last_error()
