"""Refusals of the calls that autograd records, which come before any device is asked: no GPU is needed."""
import pytest
import torch

from chimere_amd import routing

PAIRS = routing.SortedPairs(torch.arange(8, dtype=torch.int32), torch.arange(8, dtype=torch.int32).view(4, 2), torch.tensor([0, 8], dtype=torch.int32))


@pytest.mark.parametrize("grad", [False, True])
def test_scales_of_float_tokens(grad):
    """Refused with a gradient as without."""
    x = torch.randn(4, 16).requires_grad_(grad)
    for kw in (dict(scale=torch.ones(4)), dict(out_scale=torch.ones(8)), dict(scale=torch.ones(4), out_scale=torch.ones(8))):
        with pytest.raises(ValueError, match="scales: "):
            routing.dispatch(x, PAIRS, **kw)
