"""8-bit integer products at sizes that take several launches or long rows."""
import pytest
import torch

from chimere_amd import int8
from test_gpu_int8 import gen, q_ref, weights

pytestmark = pytest.mark.gpu


def shifted(n, c, g, dev):
    """n rows of c elements, each one element on in the same memory."""
    return torch.as_strided(torch.randn(n + c, generator=g, device=dev), (n, c), (1, 1))


def test_quantize_many_long_rows(dev):
    """2^24 + 3 rows that take a work-group each: more threads than one grid has."""
    n, c = (1 << 24) + 3, 1025
    print(f"quantize {n}x{c}", flush=True)
    g = gen(6)
    x = shifted(n, c, g, dev)
    q = torch.empty(n, 1040, dtype=torch.int8, device=dev)[:, :c]
    _, s = int8.quantize_i8(x, q, torch.full((n,), -1.0, device=dev))
    assert bool((s > 0).all())
    at = torch.cat([torch.tensor([0, (1 << 22) - 1, 1 << 22, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, n - 1], device=dev),
                    torch.randint(0, n, (200,), generator=g, device=dev)])
    rq, rs = q_ref(x[at])
    assert (q[at].double().cpu() == rq).all() and (s[at].double().cpu() == rs).all()


def test_linear_many_long_rows(dev):
    """The same rows through a product: as the quantizer and the product of a few of them."""
    n, c = (1 << 24) + 3, 1040
    print(f"linear {n}x1x{c}", flush=True)
    g = gen(7)
    x = shifted(n, c, g, dev)
    w, ws = weights(1, c, g)
    out = int8.linear_i8(x, w, ws)
    for first in (0, (1 << 22) - 50, (1 << 24) - 50, n - 100):
        assert torch.equal(out[first:first + 100], int8.linear_i8(x[first:first + 100], w, ws)), first
    assert bool(out.isfinite().all())


def test_quantize_longest_row(dev):
    """One row of 2^31 - 8192 columns, the most that a row may have."""
    c = 2**31 - 8192
    print(f"quantize 1x{c}", flush=True)
    x = torch.ones(1, c, dtype=torch.bfloat16, device=dev)
    x[0, -3000:] = torch.randn(3000, generator=gen(8), device=dev).to(x.dtype)
    x[0, 7] = 9.0
    q, s = int8.quantize_i8(x)
    rq, rs = q_ref(torch.cat([x[:, :64], x[:, -3000:]], 1))
    assert (s.double().cpu() == rs).all()
    assert (q[:, :64].double().cpu() == rq[:, :64]).all() and (q[:, -3000:].double().cpu() == rq[:, 64:]).all()
    assert int(q[0, 64:-3000].min()) == int(q[0, 64:-3000].max()) == int(rq[0, 0])
