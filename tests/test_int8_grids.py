"""Which sizes of the experts' call make launches of 2^32 threads or more: refused, its workspace size 0 (no GPU is needed)."""
import ctypes as C

import pytest

from chimere_amd import _lib


def accepted(H, F, E, K, T):
    layer = _lib.MoeI8LayerC(H, F, E, *[0x1000] * 6)
    return _lib.lib().chimere_moe_i8_workspace_size(C.byref(layer), K, T) > 0


def threads(H, F, E, K, T):
    """Of the larger of the two tile launches: a tile of 64 or 128 pairs per expert and block of 64 of F's or 128 of H's rows."""
    P = T * K
    rows = 64 if P / E <= 40 else 128
    tiles = P // rows + min(P, E)
    return -(-tiles * max(-(-F // 64), -(-H // 128)) // 8) * 8 * 4 * rows


@pytest.mark.parametrize("H,F,E,K", [(16, 131056, 1024, 1), (112, 87312, 1024, 1), (2048, 512, 256, 8), (64, 65536, 8, 2),
                                     (16384, 64, 1024, 16), (4096, 14336, 8, 2)])
def test_last_accepted(H, F, E, K):
    """The largest number of tokens that is taken, and one more: on the two sides of 2^32 threads or of the stated limits."""
    lo, hi = 1, 2**24
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if accepted(H, F, E, K, mid) else (lo, mid)
    assert threads(H, F, E, K, lo) < 2**32
    assert threads(H, F, E, K, hi) >= 2**32 or hi * K >= 2**24 or hi * H >= 2**31
