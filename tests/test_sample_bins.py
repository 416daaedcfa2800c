"""Host-side emulation of the bins of the first sampling launch (k_sample_scan in chimere_amd/csrc/sample.hip): the byte at
which every logit of a chunk adds to the histogram in LDS, by the kernel's own arithmetic -- the fma that rounds a logit's
octaves to an integer, of which the low 32 bits are kept -- lies inside the histogram and is the bin of the logit's level, for
masks of any finite value, at all temperatures.  The formulas are transcribed from the kernel."""
import ctypes
import math
import random

import numpy as np
import pytest

fma = ctypes.CDLL("libm.so.6").fma
fma.restype, fma.argtypes = ctypes.c_double, [ctypes.c_double] * 3

MAGIC, TABLE, BINS = 6755399441055744.0, 128, 1024
NEAR_PER, FAR = 1e-30, 2.0 ** 21
LOWEST = -3.402823466e38
END = 8 * (BINS - 1)


def low_word(m):
    b = int(np.float64(m).view(np.uint64)) & 0xFFFFFFFF
    return b - (1 << 32) if b >> 31 else b


def f32(v):
    with np.errstate(over="ignore"):
        return float(np.float32(v))


def scan_bins(logits, t, bits, counts, wave_least=LOWEST):
    """[(logit, byte)] of what the chunk's logits add to the histogram, or None where the chunk has none; counts: the branch
    that counts logits (top_k), where lanes may leave out what is below `wave_least`; else the one that adds weights."""
    top = max(logits)
    per = 1.44269504088896340736 * TABLE / f32(t)
    if not (per >= NEAR_PER and abs(top * per) < FAR * TABLE):
        return None
    k = low_word(fma(top, per, MAGIC))
    less = (k >> 7) + 1
    magic = MAGIC + TABLE * float(bits - less)
    low = (k + TABLE * (bits - less)) & ~7
    least = f32((k - 70 * TABLE) / per)
    if counts:
        least = max(least, LOWEST, wave_least)
    out = []
    for x in logits:
        if x >= least:
            at = low - (low_word(fma(x, per, magic)) & ~7)
            assert -2 ** 31 <= at < 2 ** 31     # (no signed overflow)
            out.append((x, min(at, END)))
    return out


def check(logits, t, bits, counts, **kw):
    got = scan_bins(logits, t, bits, counts, **kw)
    if got is None:
        return 0
    per = 1.44269504088896340736 * TABLE / f32(t)
    top = max(logits)
    for x, at in got:
        assert 0 <= at <= END and at % 8 == 0, (x, at, t)
        octaves = (top - x) * per / 8 / 16      # below the largest
        assert abs(at / 8 - 16 * octaves) <= 1.5 or at == END and octaves > 63, (x, at, t)
    assert {x for x, _ in got} >= {x for x in logits if (top - x) * per < 60 * TABLE and x >= kw.get("wave_least", LOWEST)}
    return len(got)


TEMPERATURES = [0.380492598, 0.25, 0.5, 0.6, 0.8, 1.0, 1.2, 1.7, 2.0, 1e-3, 100.0, 1e5, 7.21000033e-05, 1e-7, 3e30]
MASKS = [-1e4, -1e5, -1e6, -1e7, -1e8, -1e9, -1e10, -1e15, -1e20, -1e30, -65504.0, LOWEST, -3.3895314e38]
TOPS = [20.0, 0.0, -3.25, 11.4375, 88.8, 65504.0, -1e9, 3e5, LOWEST]


@pytest.mark.parametrize("counts", [True, False])
@pytest.mark.parametrize("bits", [42, 44, 47, 51])
def test_bins_of_masked_rows(bits, counts):
    rng = random.Random(bits)
    seen = 0
    for t in TEMPERATURES + [rng.uniform(0.25, 2.0) for _ in range(60)] + [10.0 ** rng.uniform(-6, 6) for _ in range(20)]:
        for top in TOPS:
            top = f32(top)
            for mask in MASKS:
                x = [top, f32(top - 0.5 * t), f32(top - 5 * t), f32(top - 30 * t), f32(top - 69 * t), f32(top - 71 * t), f32(min(mask, top))]
                seen += check([v for v in x if math.isfinite(v)], t, bits, counts)
    assert seen > 4000


def test_bins_of_waves_that_leave_out(bits=44):
    """A wave whose lanes all have something above the mask leaves out the rest; one with a masked lane does not."""
    x = [20.0, 19.0, 3.0, -1e9, LOWEST]
    for t in TEMPERATURES:
        for least in (3.0, -1e9, LOWEST):
            check(x, t, bits, True, wave_least=least)
