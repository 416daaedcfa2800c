"""Cuts and sums of rows in chunks of 16384 logits, where they could disagree: against the definition in 64 bits, as
tests/test_gpu_sampling.py does it, with outputs that are filled before the call, so that a token that is not written shows."""
import pytest
import torch

from chimere_amd import sampling
from test_gpu_sampling import TYPES, check, logits

pytestmark = pytest.mark.gpu


def filled(n, dev):
    return {"out": torch.full((n,), -77, dtype=torch.int32, device=dev), "logprob": torch.full((n,), 77.0, device=dev)}


@pytest.mark.parametrize("top,t", [(29.0481281, 7.21000033e-05), (30.9268703, 7.56000081e-05), (26.7155972, 4.51999986e-05)])
def test_min_p_of_one_ends_at_the_largest(dev, top, t):
    """The largest logit's octaves lie just below a border between two bins, where they are rounded."""
    print(f"sample min_p=1 top={top} T={t}", flush=True)
    x = torch.zeros(3, 20000, device=dev)
    x[:, 5] = top
    x[1, [5, 19000]] = x[1, [19000, 5]]
    x[2, 19999] = top
    for p in (1.0, 0.5):
        token, logprob = sampling.sample(x, torch.tensor([0.5, 0.5, 0.75], device=dev), temperature=t, top_p=p, min_p=1.0, **filled(3, dev))
        assert token.tolist() == [5, 19000, 19999 if p == 1 else 5]
        assert logprob.tolist()[:2] == [0.0, 0.0] and abs(logprob[2].item() + (0.6931472 if p == 1 else 0.0)) < 1e-6


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [20000, 151936])
def test_min_p(dev, V, dtype):
    """min_p alone and with a share, from the largest logit's equals to nearly all, warm and cold."""
    g = torch.Generator(device="cuda").manual_seed(V)
    for kind in ("power", "flat", "peak", "wide"):
        x = logits(kind, 8, V, g, dev).to(TYPES[dtype])
        u = torch.rand(8, generator=g, device=dev).clamp(1e-3, 1 - 1e-3)
        for m in (1.0, 1 - 2.0 ** -24, 0.6, 0.05, 1e-3, 1e-12):
            for t, p in ((1.0, 1.0), (0.05, 1.0), (2.5, 0.97), (1e-4, 1.0)):
                print(f"sample V={V} {kind} {dtype} min_p={m} T={t} top_p={p}", flush=True)
                check(x, u, temperature=t, top_p=p, min_p=m, undecided=0.25, **filled(8, dev))
