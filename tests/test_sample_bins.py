"""Host-side emulation of the bins of the sampling launches: that of the first one (k_sample_scan in chimere_amd/csrc/sample.hip): the byte at
which every logit of a chunk adds to the histogram in LDS, by the kernel's own arithmetic -- the fma that rounds a logit's
octaves to an integer, of which the low 32 bits are kept -- lies inside the histogram and is the bin of the logit's level, for
masks of any finite value, at all temperatures; and, of the second (k_sample_pick), the bin that min_p ends in, which is found
from the first logit that is at least min_p of the largest: never above the largest logit's own.  The formulas are transcribed
from the kernels."""
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


def logit_key(x):
    b = int(np.float32(x + 0.0).view(np.uint32))
    return ~b & 0xFFFFFFFF if b >> 31 else b | 0x80000000


def key_logit(k):
    return float(np.uint32(k & 0x7FFFFFFF if k >> 31 else ~k & 0xFFFFFFFF).view(np.float32))


TABLE_POWERS = [math.exp(math.log(2) * (j / 128 - 0.5)) * 2 ** 0.5 for j in range(128)]


def real(x, top, per):
    """The probability of x relative to that of the largest."""
    if x == top:
        return 1.0
    d = max(x - top, -min(2.0 ** 30 / per, 2.0 ** 1000))
    m = fma(d, per, MAGIC)
    k, f = low_word(m), fma(d, per, MAGIC - m)
    if k < -1000 * TABLE:
        return 0.0
    L = math.log(2) / TABLE
    p = 1.0
    for c in (L ** 4 / 24, L ** 3 / 6, L ** 2 / 2, L, 1.0):
        p = c if c == L ** 4 / 24 else fma(p, f, c)
    return math.ldexp(TABLE_POWERS[k & 127] * p, k >> 7)


def least_start(top, per, least):
    below = TABLE * math.log2(least) / per
    v = top + below
    far = abs(v) * 1e-6 + (abs(top) - below) * 1e-12 + 1e-9 / per
    lo, hi = logit_key(f32(max(v - far, LOWEST))) - 1, min(logit_key(f32(min(v + far, top))), logit_key(top))
    assert real(key_logit(lo), top, per) < least or key_logit(lo) < LOWEST or key_logit(lo) == -math.inf
    assert real(key_logit(hi), top, per) >= least
    while hi - lo > 1:
        step = (hi - lo + 63) // 64
        f = next(i for i in range(64) if min(lo + (i + 1) * step, hi) == hi or real(key_logit(min(lo + (i + 1) * step, hi)), top, per) >= least)
        lo, hi = lo + f * step, min(lo + (f + 1) * step, hi)
    return hi


def level(x, per, magic):
    return low_word(fma(x, per, magic)) >> 3


def test_bin_of_min_p():
    rng = random.Random(3)
    cases = [(29.0481281, 7.21000033e-05, 1.0), (30.9268703, 7.56000081e-05, 1.0), (26.7155972, 4.51999986e-05, 1.0)]
    for _ in range(3000):
        t, top = 10.0 ** rng.uniform(-5, 5), rng.choice([-1, 1]) * 10.0 ** rng.uniform(-6, 4)
        cases.append((rng.choice([top, 0.0, 11.5 * t]), t, rng.choice([1.0, 1 - 2.0 ** -24, 0.5, 0.1, 10.0 ** rng.uniform(-12, 0), 1e-45])))
    seen = 0
    for top, t, least in cases:
        top, t, least = f32(top), f32(t), f32(least)
        per = 1.44269504088896340736 * TABLE / t
        if not abs(top * per) < 2.0 ** 20 * TABLE:
            continue
        seen += 1
        less = (low_word(fma(top, per, MAGIC)) >> 7) + 1
        magic = MAGIC + TABLE * float(47 - less)
        key = least_start(top, per, least)
        low = level(top, per, magic) - level(key_logit(key), per, magic)
        assert low >= 0 and (low == 0 or least < 1), (top, t, least, low)
        assert abs(low + 16 * math.log2(least)) <= 1.01, (top, t, least, low)
        # from the key on the probability is that, below it is not (but for the last places of the reference's own)
        assert (key_logit(key) - top) / t >= math.log(least) - 1e-11, (top, t, least)
        assert (key_logit(key - 1) - top) / t < math.log(least) + 1e-11, (top, t, least)
    assert seen > 1000
