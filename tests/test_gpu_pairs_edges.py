"""Sorted pairs at the edges of what may be called: no tokens in 8 bits, too many experts."""
import pytest
import torch

from chimere_amd import routing
from chimere_amd._lib import ChimereError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [32, 5000])
def test_no_tokens_in_8_bits(dev, cols):
    """Rows behind the last pair, of an out that has some: cleared with their scales."""
    pairs = routing.sort_pairs(torch.empty(0, 4, dtype=torch.int32, device=dev), 9)
    q = torch.empty(0, cols, dtype=torch.int8, device=dev)
    out = torch.full((3, (cols + 15) // 16 * 16), 2, dtype=torch.int8, device=dev)[:, :cols]
    scale = torch.full((3,), float("nan"), device=dev)
    rows, scales = routing.dispatch(q, pairs, scale=torch.empty(0, device=dev), out=out, out_scale=scale)
    assert rows is out and scales is scale and (rows == 0).all() and scales.tolist() == [0.0] * 3
    assert routing.dispatch(q, pairs, scale=torch.empty(0, device=dev), out=out)[1].tolist() == [0.0] * 3
    rows, scales = routing.dispatch(q, pairs, scale=torch.empty(0, device=dev))
    assert rows.shape == (0, cols) and scales.shape == (0,)


def test_experts_past_the_most(dev):
    """Refused before anything of their number is allocated."""
    ids = torch.tensor([[0, 1], [1023, -1]], dtype=torch.int32, device=dev)
    assert routing.sort_pairs(ids, 1024).offsets.tolist() == [0, 1] + [2] * 1022 + [3]
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for n in (1025, 10 ** 6, 10 ** 8):
        with pytest.raises(ChimereError) as e:
            routing.sort_pairs(ids, n)
        assert e.value.code == 1 and f"n_experts={n} " in str(e.value)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
