"""Sizes past what the 8-bit integer and balance-loss calls count in: refused before a launch, so no GPU is needed."""
import ctypes as C

import pytest
import torch

from chimere_amd import _lib, int8, routing

P = C.c_void_p(0x1000)      # aligned, never read
LONGEST = 2**31 - 8192      # columns of a quantized row
FAR = 2**32 + 64            # as a C int: 64


def quantize(nrows, ncols):
    _lib.lib().chimere_quantize_i8(1, P, ncols, P, 1 << 31, P, nrows, ncols, None)
    return _lib.lib().chimere_hip_get_last_error(), _lib.lib().chimere_hip_get_last_error_string().decode()


@pytest.mark.parametrize("ncols", [LONGEST + 1, 2**31 - 1024, 2**31 - 1])
def test_rows_whose_columns_would_overflow(ncols):
    """A thread counts columns in int, 2048 at a time past the last."""
    code, msg = quantize(1, ncols)
    assert code == 1 and "ncols" in msg
    assert quantize(0, LONGEST)[0] == 0


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("call", [
    lambda: int8.quantize_i8(meta(1, FAR)),
    lambda: int8.quantize_i8(meta(FAR, 4)),
    lambda: int8.linear_i8(meta(1, FAR), meta(4, FAR, dtype=torch.int8), meta(4)),
    lambda: int8.linear_i8(meta(FAR, 64), meta(4, 64, dtype=torch.int8), meta(4)),
    lambda: int8.linear_i8(meta(4, 64), meta(FAR, 64, dtype=torch.int8), meta(FAR)),
    lambda: int8.gemm_i8(meta(FAR, 64, dtype=torch.int8), meta(FAR), meta(4, 64, dtype=torch.int8), meta(4)),
    lambda: int8.gemm_i8(meta(4, 64, dtype=torch.int8), meta(4), meta(4, 64, dtype=torch.int8), meta(4), out=meta(FAR, 4)),
    lambda: int8.Int8Experts(*(meta(*s, dtype=d) for s, d in (
        ((1, FAR, 16), torch.int8), ((1, FAR), torch.float32), ((1, FAR, 16), torch.int8), ((1, FAR), torch.float32),
        ((1, 16, FAR), torch.int8), ((1, 16), torch.float32)))),
    lambda: routing.balance_loss(meta(FAR, 4), meta(FAR, 2, dtype=torch.int32)),
    lambda: routing.balance_loss(meta(4, 8), meta(4, FAR, dtype=torch.int32)),
    lambda: routing.balance_loss_grad(meta(4, 8), meta(8, dtype=torch.int32), meta(1, dtype=torch.int32), meta(1), FAR),
])
def test_sizes_past_int32(call):
    """The C entry points take these as int: 2^32 + 64 would be 64."""
    with pytest.raises(ValueError, match="2147483647"):
        call()
