"""The layer norm's C entries take row statistics in 16-byte rows and refuse a
pointer that is not aligned to them, before anything is launched.  No GPU needed."""

import ctypes

import pytest

from theria_b200 import _lib

P = ctypes.c_void_p(16)  # never dereferenced: validation fails first


@pytest.mark.parametrize("offset", [4, 8])
def test_misaligned_statistics_are_refused(offset):
    lib, stats = _lib.load(), ctypes.c_void_p(16 + offset)
    assert lib.theria_norm_fwd(P, P, P, 0, P, stats, 4, 16, 0, 1e-5, None) \
        == _lib.THERIA_ERR_INVALID_ARG
    assert lib.theria_norm_bwd(P, P, 0, P, stats, P, None, None, None, 0, 4, 16, 0, None) \
        == _lib.THERIA_ERR_INVALID_ARG
    assert lib.theria_norm_bwd2(P, P, 0, P, stats, P, P, P, P, P, P, P, 1 << 20, 4, 16, 0, None) \
        == _lib.THERIA_ERR_INVALID_ARG
