"""Refusals of the calls that autograd records, which come before any device is asked: no GPU is needed."""
import pytest
import torch
from torch.autograd import forward_ad

from chimere_amd import norm, routing

PAIRS = routing.SortedPairs(torch.arange(8, dtype=torch.int32), torch.arange(8, dtype=torch.int32).view(4, 2), torch.tensor([0, 8], dtype=torch.int32))


@pytest.mark.parametrize("grad", [False, True])
def test_scales_of_float_tokens(grad):
    """Refused with a gradient as without."""
    x = torch.randn(4, 16).requires_grad_(grad)
    for kw in (dict(scale=torch.ones(4)), dict(out_scale=torch.ones(8)), dict(scale=torch.ones(4), out_scale=torch.ones(8))):
        with pytest.raises(ValueError, match="scales: "):
            routing.dispatch(x, PAIRS, **kw)


@pytest.mark.parametrize("grad", [False, True])
def test_tangents(grad):
    """A tangent would be lost: refused, with a gradient recorded beside it or not; the same values without one pass on to the
    checks of the call itself."""
    x, y, w = torch.randn(4, 16), torch.randn(8, 16), torch.rand(4, 2)
    ids, weight = torch.zeros(4, 2, dtype=torch.int32), torch.randn(16)
    calls = [(lambda t: norm.rms_norm(t), x), (lambda t: norm.rms_norm(x, t), weight), (lambda t: norm.rms_norm(x, weight, residual=t), x),
             (lambda t: routing.dispatch(t, PAIRS), x), (lambda t: routing.combine(t, PAIRS, w), y), (lambda t: routing.combine(y, PAIRS, t), w),
             (lambda t: routing.balance_loss(t, ids), x)]
    for call, t in calls:
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="tangent"):
                call(forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t)))
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call(forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t)))
            with pytest.raises(ValueError, match="ROCm device"):
                call(t.clone().requires_grad_(grad))
        with pytest.raises(ValueError, match="ROCm device"):
            call(t.clone().requires_grad_(grad))
