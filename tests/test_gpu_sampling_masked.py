"""Sampling from rows of which nearly all is masked by a finite number, by top-k: against the definition in 64 bits, as
tests/test_gpu_sampling.py does it.  A mask's logits weigh nothing, whatever the temperature, and may not come into the count
of the first top_k by another bin than their own."""
import pytest
import torch

from test_gpu_sampling import TYPES, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [-1e7, -1e9, -1e10, "lowest"])
@pytest.mark.parametrize("V", [20000, 151936])
def test_top_k_of_masked_rows(dev, V, mask, dtype):
    """Half a per cent and a hundredth of a per cent stay (a wave's lanes then have masked logits alone); the largest is 20."""
    g = torch.Generator(device="cuda").manual_seed(V)
    n, fin = 6, torch.finfo(TYPES[dtype])
    low = fin.min if mask == "lowest" else max(mask, fin.min)
    x = 4 * torch.randn(n, V, generator=g, device=dev)
    x[torch.arange(n), torch.randint(0, V, (n,), generator=g, device=dev)] = 20.0
    keep = torch.rand(n, V, generator=g, device=dev) < torch.tensor([[5e-3], [1e-4]] * (n // 2), device=dev)
    x = torch.where(keep | (x == 20.0), x.clamp(max=20.0), torch.full_like(x, low)).to(TYPES[dtype])
    u = torch.rand(n, generator=g, device=dev).clamp(1e-3, 1 - 1e-3)
    for t in (0.380492598, 0.5, 0.6, 0.8, 1.0, 1.2):
        for k in (20, 64, 100, 1000):
            print(f"sample masked V={V} mask={low} {dtype} T={t} top_k={k}", flush=True)
            token, _ = check(x, u, temperature=t, top_k=k)
            assert (x.float()[torch.arange(n, device=dev), token.long()] > low).all()
