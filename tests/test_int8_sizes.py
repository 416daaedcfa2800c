"""Sizes past what the 8-bit integer calls count in: refused before a launch, so no GPU is needed."""
import ctypes as C

import pytest

from chimere_amd import _lib

P = C.c_void_p(0x1000)      # aligned, never read
LONGEST = 2**31 - 8192      # columns of a quantized row


def quantize(nrows, ncols):
    _lib.lib().chimere_quantize_i8(1, P, ncols, P, 1 << 31, P, nrows, ncols, None)
    return _lib.lib().chimere_hip_get_last_error(), _lib.lib().chimere_hip_get_last_error_string().decode()


@pytest.mark.parametrize("ncols", [LONGEST + 1, 2**31 - 1024, 2**31 - 1])
def test_rows_whose_columns_would_overflow(ncols):
    """A thread counts columns in int, 2048 at a time past the last."""
    code, msg = quantize(1, ncols)
    assert code == 1 and "ncols" in msg
    assert quantize(0, LONGEST)[0] == 0
