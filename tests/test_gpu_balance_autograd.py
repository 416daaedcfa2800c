"""The balance loss within a program's own backward pass: its gradient is that of ``balance_loss_grad``, bit for bit, whose
own tolerances against 64 bits stand in test_gpu_balance.py."""
import pytest
import torch

from chimere_amd import routing
from test_gpu_balance import STEP, TYPES, U, choice, ref

pytestmark = pytest.mark.gpu


def plain(logits, ids, g, mask=None):
    """The gradient by the two plain calls."""
    x = logits.detach()
    _, counts, _, tokens = routing.balance_loss(x, ids, mask=mask)
    return routing.balance_loss_grad(x, counts, tokens, torch.full((1,), g, device=x.device), ids.shape[1], mask=mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,K", [(0, 8, 2), (1, 1, 1), (7, 65, 4), (300, 256, 8), (1025, 600, 3)])
def test_backward(dev, T, E, K, dtype):
    print(f"balance backward T={T} E={E} K={K} {dtype}", flush=True)
    x, ids, g = choice(T, E, K, T + E, TYPES[dtype], dev, drop=0.1)
    mask = torch.rand(T, generator=g, device=dev) < 0.6
    for m in (None, mask):
        leaf = x.clone().requires_grad_()
        loss, counts, probs, tokens = routing.balance_loss(leaf, ids, mask=m)
        assert loss.requires_grad and not (counts.requires_grad or probs.requires_grad or tokens.requires_grad)
        assert all(torch.equal(a, b) for a, b in zip((loss, counts, probs, tokens), routing.balance_loss(x, ids, mask=m)))
        (0.25 * loss).sum().backward()
        assert leaf.grad.dtype == x.dtype and torch.equal(leaf.grad, plain(x, ids, 0.25, m))


def test_next_to_another_loss(dev):
    """Added to another loss, neither term is dropped; logits that are no leaf, rows apart."""
    T, E, K = 130, 96, 4
    w = torch.randn(T, E + 7, device=dev, requires_grad=True)
    ids = choice(T, E, K, 3, torch.float32, dev)[1]
    logits = (2 * w)[:, 3:3 + E]
    other = logits.square().sum()
    (other + 0.5 * routing.balance_loss(logits, ids)[0]).sum().backward()
    want = torch.zeros_like(w)
    want[:, 3:3 + E] = 2 * (2 * logits.detach() + plain(logits, ids, 0.5))
    # two sums of the same two terms: half a step each
    assert bool(((w.grad - want).abs() <= 4 * U * want.abs() + 2.0 ** -149).all())
    assert not torch.equal(w.grad[:, 3:3 + E], (4 * logits).detach())


def test_the_formula_in_64_bits(dev):
    """Against torch's own differentiation of the formula in 64 bits, counts held."""
    T, E, K = 90, 40, 3
    x, ids, _ = choice(T, E, K, 5, torch.float32, dev)
    leaf = x.clone().requires_grad_()
    loss, counts, _, _ = routing.balance_loss(leaf, ids)
    loss.backward()
    v = x.double().cpu().requires_grad_()
    (E * (counts.double().cpu() / (T * K) * torch.softmax(v, 1).mean(0)).sum()).backward()
    _, (_, _, tol) = ref(x, ids, None, 1.0)
    assert bool(((leaf.grad.double().cpu() - v.grad).abs() <= tol).all())


def test_scaled_loss_in_16_bits(dev):
    """The gradient has the logits' type: in f16 most of a training step's is under its smallest number, and a scaled loss
    (as any training in f16 has) keeps it: 2^16 times, exact but for the type's own rounding."""
    T, E, K = 4000, 64, 4
    x, ids, _ = choice(T, E, K, 6, torch.float16, dev)
    small, large = x.clone().requires_grad_(), x.clone().requires_grad_()
    (0.01 * routing.balance_loss(small, ids)[0]).backward()
    (0.01 * 2.0 ** 16 * routing.balance_loss(large, ids)[0]).backward()
    assert float((small.grad == 0).float().mean()) > 0.5 and float((large.grad == 0).float().mean()) < 0.1
    (_, _, _, _, want), (_, _, tol) = ref(x, ids, None, float(torch.tensor(0.01 * 2.0 ** 16)))
    assert bool(((large.grad.double().cpu() - want).abs() <= tol + 2 * STEP[x.dtype] * U * want.abs()).all())


def test_what_is_not_recorded(dev):
    x, ids, _ = choice(20, 16, 2, 1, torch.float32, dev)
    leaf = x.clone().requires_grad_()
    with torch.no_grad():
        assert not routing.balance_loss(leaf, ids)[0].requires_grad
    assert not routing.balance_loss(leaf.detach(), ids)[0].requires_grad
    loss = routing.balance_loss(leaf, ids)[0]
    grad, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):                       # a second derivative
        grad.sum().backward()
    loss = routing.balance_loss(leaf * 1, ids)[0]
    moved = leaf * 1
    loss = routing.balance_loss(moved, ids)[0]
    moved.add_(1)
    with pytest.raises(RuntimeError):                       # logits that were changed in between
        loss.backward()
    with pytest.raises(ValueError):
        routing.balance_loss(leaf, ids.long())


def test_captured(dev):
    """Forward and backward in one graph, replayed on new logits with eager calls of another leaf between."""
    T, E, K = 300, 64, 4
    x, ids, g = choice(T, E, K, 9, torch.float32, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = x.clone().requires_grad_()
        torch.autograd.grad(routing.balance_loss(warm, ids)[0], warm)
        del warm
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    leaf = x.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = routing.balance_loss(leaf, ids)[0]
        grad, = torch.autograd.grad(0.5 * loss, leaf)
    for i in range(4):
        print(f"balance backward replay {i}", flush=True)
        with torch.no_grad():
            leaf.copy_(torch.randn(T, E, generator=g, device=dev))
        graph.replay()
        want = plain(leaf, ids, 0.5)
        torch.cuda.synchronize()
        assert torch.equal(grad, want) and torch.equal(loss.detach(), routing.balance_loss(leaf.detach(), ids)[0])
