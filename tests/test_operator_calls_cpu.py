"""Refusals and host-side behaviour of the operators around the block that need
no GPU."""
import ctypes

import pytest

from swiglu_b200 import _lib

P = 256
TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _refused(lib, rc, text):
    assert rc == 1 and text in lib.swiglu_b200_last_error_message(), (rc, lib.swiglu_b200_last_error_message())


@pytest.mark.parametrize("cols", [TOP, TOP - 1023])
def test_norm_rows_whose_column_numbers_would_overflow(lib, cols):
    """The looping kernels add up to 1024 to an int column number: past
    2^31 - 1025 columns it would turn negative inside the row."""
    eps = ctypes.byref(ctypes.c_float(1e-6))
    n = ctypes.c_int64(0)
    _refused(lib, lib.swiglu_b200_rmsnorm_fwd(P, P, P, P, P, P, 1, cols, eps, 1, 1, None), b"at most 2147482623 columns")
    _refused(lib, lib.swiglu_b200_rmsnorm_fwd_e4m3(P, P, P, P, P, P, P, 1, cols, eps, 1, 1, None), b"at most")
    _refused(lib, lib.swiglu_b200_rmsnorm_bwd(P, P, P, P, P, P, P, P, 1 << 40, 1, cols, 1, 1, None), b"at most")
    _refused(lib, lib.swiglu_b200_rmsnorm_bwd_workspace(1, cols, 148, ctypes.byref(n)), b"at most")
    assert lib.swiglu_b200_rmsnorm_bwd_workspace(1, TOP - 1024, 148, ctypes.byref(n)) == 0
