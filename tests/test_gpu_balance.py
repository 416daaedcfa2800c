"""Balance loss, per-expert counts and the gradient of the logits against a
plain form in 64 bits, and the gradient against differences.

Tolerances, u = 2^-24: a probability's relative error is at most
(|x - max| + 30) u: the rounding of x - max (|x - max| u), the exponential
(2 u), the row's sum (at most 16 terms in a lane and 6 levels), the reciprocal
and a product.  Sums over tokens add at most one rounding per addition (rows
of a wave, 4 waves, at most 1024 groups).  Counts are equal."""
import pytest
import torch

from chimere_amd import ggml_gpu as G
from chimere_amd import routing
from chimere_amd._lib import ChimereError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def ref(logits, ids, mask, g):
    """(loss, counts, probs, tokens, grad) and the tolerances of loss, probs and grad, in 64 bits on the CPU."""
    x, ids = logits.double().cpu(), ids.cpu().long()
    T, E = x.shape
    K = ids.shape[1]
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu().bool()
    n = int(keep.sum())
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    none = (x == -float("inf")).all(1)
    m = torch.where(none, torch.zeros(T, dtype=torch.float64), x.amax(1)) if T else x.new_zeros(0)
    e = torch.exp(x - m[:, None])
    s = e.sum(1, keepdim=True)
    p = torch.where(s > 0, e / s, torch.zeros_like(e)) * keep[:, None]
    inside = keep[:, None] & (ids >= 0) & (ids < E)
    counts = torch.bincount(ids[inside], minlength=E)
    f = counts.double() / max(n * K, 1)
    P = p.sum(0) / max(n, 1)
    d = (p @ f)[:, None]
    c = abs(g) * E / max(n, 1)
    loss, grad = E * (f @ P), g * E / max(n, 1) * p * (f - d)
    # an exponential below e^-86 is 0 in the kernel
    rel = torch.where(p > 0, ((x - m[:, None]).abs() + 30) * U, torch.zeros_like(p))
    tp = (p * rel + torch.where(p < 1e-36, p, torch.zeros_like(p)) + 2.0 ** -149)
    adds = 64 + 4 + 1024
    tol_P = tp.sum(0) / max(n, 1) + (adds + 2) * U * P
    tol_loss = E * (f @ tol_P) + (16 + 20) * U * loss
    tol_grad = c * (tp * (f - d).abs() + p * ((tp @ f)[:, None] + (f + d) * 30 * U)) + 6 * U * grad.abs()
    dt = logits.dtype
    return (loss, counts, P, n, grad), (tol_loss, tol_P, tol_grad * (1 + STEP[dt]) + STEP[dt] * grad.abs() + TINY[dt])


def check(logits, ids, mask=None, g=0.7, out=None):
    loss, counts, probs, tokens = routing.balance_loss(logits, ids, mask=mask)
    gl = torch.full((1,), g, device=logits.device)
    grad = routing.balance_loss_grad(logits, counts, tokens, gl, ids.shape[1], mask=mask, out=out)
    torch.cuda.synchronize()
    g = float(gl)
    (rl, rc, rp, rn, rg), (tl, tp, tg) = ref(logits, ids, mask, g)
    assert int(tokens) == rn and (counts.cpu().long() == rc).all()
    assert ((probs.double().cpu() - rp).abs() <= tp).all(), (probs.double().cpu() - rp).abs().max()
    assert abs(float(loss) - float(rl)) <= float(tl), (float(loss), float(rl), float(tl))
    bad = (grad.double().cpu() - rg).abs() > tg
    assert not bad.any(), ((grad.double().cpu() - rg)[bad][:4], tg[bad][:4])
    return loss, counts, probs, tokens, grad


def choice(T, E, K, seed, dtype, dev, drop=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (2 * torch.randn(T, E, generator=g, device=dev)).to(dtype)
    ids = torch.rand(T, E, generator=g, device=dev).topk(K, dim=1)[1].to(torch.int32)
    ids[torch.rand(T, K, generator=g, device=dev) < drop] = -1
    return x, ids, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 256, 8), (2, 3, 2), (5, 64, 6), (7, 65, 4), (33, 100, 3), (64, 256, 8), (63, 200, 8),
                                   (257, 256, 8), (300, 1024, 10), (1000, 257, 2), (1023, 8, 2), (1024, 128, 8), (1025, 255, 5),
                                   (3000, 512, 4), (5000, 60, 6), (9001, 256, 8), (20000, 24, 4), (64, 1023, 8), (65, 645, 4), (219, 645, 4), (4200, 600, 2),
                                   (257, 13, 2), (16500, 513, 3)])
def test_balance(dev, T, E, K, dtype):
    print(f"balance T={T} E={E} K={K} {dtype}", flush=True)
    x, ids, g = choice(T, E, K, T + E, TYPES[dtype], dev, drop=0.1)
    check(x, ids)
    check(x, ids, mask=torch.rand(T, generator=g, device=dev) < 0.6)


@pytest.mark.parametrize("T,E,K", [(257, 16, 2), (260, 33, 3), (300, 64, 4), (513, 64, 4), (300, 128, 8), (600, 256, 8), (600, 511, 8),
                                   (2048, 256, 2), (2049, 256, 2), (8192, 256, 2), (8193, 253, 2), (128, 512, 8), (33, 1021, 4),
                                   (128, 1024, 8), (512, 1024, 2), (513, 1024, 2), (4096, 7, 1), (4097, 7, 1), (70000, 5, 2)])
def test_balance_joins(dev, T, E, K):
    """Sizes on both sides of where the work is shared out another way."""
    print(f"balance joins T={T} E={E} K={K}", flush=True)
    x, ids, g = choice(T, E, K, T * E, torch.bfloat16, dev, drop=0.1)
    first = check(x, ids)
    again = routing.balance_loss(x, ids)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 9, 130, 2000])
def test_masks_and_odd_values(dev, T, dtype):
    """All tokens left out, one kept, NaN in rows left out, ids of all kinds, experts masked by -inf, rows of -inf,
    the type's lowest value, far logits, many ties."""
    x, ids, g = choice(T, 96, 4, T, TYPES[dtype], dev)
    low = float(torch.finfo(TYPES[dtype]).min)
    print(f"balance odd T={T} {dtype}", flush=True)
    none = torch.zeros(T, dtype=torch.bool, device=dev)
    _, _, _, _, grad = check(x, ids, mask=none)
    assert (grad == 0).all()
    one = none.clone()
    one[T // 2] = True
    y = torch.where(one[:, None], x, torch.full_like(x, float("nan")))
    check(y, ids, mask=one.to(torch.uint8) * 255)
    check(x, torch.randint(-5, 101, (T, 4), generator=g, device=dev).to(torch.int32))
    check(x, torch.full((T, 4), 7, dtype=torch.int32, device=dev))
    check(x, torch.full((T, 4), -1, dtype=torch.int32, device=dev))
    y = x.clone()
    y[:, 5:60] = -float("inf")
    check(y, ids)
    y[::2] = -float("inf")
    check(y, ids)
    y = x.clone()
    y[:, 3:90] = low
    check(y, ids)
    y[::2] = low
    check(y, ids)
    check((x.float() * 30).to(x.dtype), ids)
    check(torch.zeros_like(x), ids)


def test_infinity_and_nan_show(dev):
    """A NaN or +inf logit of a kept token shows in the loss and in its own row's gradient only."""
    x, ids, _ = choice(50, 64, 4, 1, torch.float32, dev)
    for v in (float("nan"), float("inf")):
        y = x.clone()
        y[7, 9] = v
        loss, counts, probs, tokens = routing.balance_loss(y, ids)
        grad = routing.balance_loss_grad(y, counts, tokens, torch.ones(1, device=dev), 4)
        assert loss.isnan().all() and grad[7].isnan().any()
        keep = torch.arange(50) != 7
        assert grad.cpu()[keep].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_what_is_left(dev, dtype):
    T, E = 70, 99
    x, ids, _ = choice(T, E + 14, 5, 3, TYPES[dtype], dev)
    ids = (ids % E).contiguous()
    room = torch.full((T, E + 9), 2.0, dtype=TYPES[dtype], device=dev)
    check(x[:, 3:3 + E], ids, out=room[:, 2:2 + E])
    assert (room[:, :2] == 2.0).all() and (room[:, 2 + E:] == 2.0).all()
    check(x[:1, 3:3 + E].expand(T, E), ids)


def test_gradient_against_differences(dev):
    """Central differences of the loss in 64 bits, counts held: step 1e-4, error below 1e-7 of the largest entry."""
    x, ids, _ = choice(6, 12, 3, 11, torch.float32, dev)
    _, counts, _, tokens = routing.balance_loss(x, ids)
    grad = routing.balance_loss_grad(x, counts, tokens, torch.ones(1, device=dev), 3).double().cpu()
    f = counts.double().cpu() / 18

    def loss(v):
        return 12 * (f @ torch.softmax(v, 1).mean(0))

    v, want = x.double().cpu(), torch.zeros(6, 12, dtype=torch.float64)
    for t in range(6):
        for j in range(12):
            step = torch.zeros_like(v)
            step[t, j] = 1e-4
            want[t, j] = (loss(v + step) - loss(v - step)) / 2e-4
    assert ((grad - want).abs() <= 1e-6 * want.abs().max() + 40 * U * 12 / 6 * (f.max() * 2)).all()


def test_repeats_and_graph(dev):
    """The same bits on every call, in a replayed graph too, with eager calls and new inputs between."""
    for T in (40, 3000):
        x, ids, g = choice(T, 256, 8, 2, torch.float32, dev)
        mask = torch.rand(T, generator=g, device=dev) < 0.8
        one, grad = torch.full((1,), 0.01, device=dev), torch.empty_like(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            routing.balance_loss(x, ids, mask=mask)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = routing.balance_loss(x, ids, mask=mask)
            routing.balance_loss_grad(x, got[1], got[3], one, 8, mask=mask, out=grad)
        for i in range(4):
            print(f"balance graph T={T} replay {i}", flush=True)
            x.copy_(torch.randn(T, 256, generator=g, device=dev))
            mask.copy_(torch.rand(T, generator=g, device=dev) < 0.5)
            graph.replay()
            want = routing.balance_loss(x, ids, mask=mask)
            wg = routing.balance_loss_grad(x, want[1], want[3], one, 8, mask=mask)
            torch.cuda.synchronize()
            assert all((a == b).all() for a, b in zip(got, want)) and (grad == wg).all()


def test_no_tokens(dev):
    x, ids = torch.empty(0, 40, device=dev), torch.empty(0, 4, dtype=torch.int32, device=dev)
    loss, counts, probs, tokens = routing.balance_loss(x, ids)
    assert float(loss) == 0 and (counts == 0).all() and (probs == 0).all() and int(tokens) == 0
    assert routing.balance_loss_grad(x, counts, tokens, loss, 4).shape == (0, 40)


def test_refusals(dev):
    x, ids, _ = choice(8, 32, 2, 1, torch.float32, dev)
    loss, counts, _, tokens = routing.balance_loss(x, ids)
    for f in (lambda: routing.balance_loss(x.double(), ids), lambda: routing.balance_loss(x.t(), ids),
              lambda: routing.balance_loss(x, ids.long()), lambda: routing.balance_loss(x, ids[:5]),
              lambda: routing.balance_loss(x, ids, mask=torch.ones(8, device=dev)),
              lambda: routing.balance_loss(x, ids, mask=torch.ones(7, dtype=torch.bool, device=dev)),
              lambda: routing.balance_loss(x, ids.cpu()), lambda: routing.balance_loss(x.cpu(), ids.cpu()),
              lambda: routing.balance_loss_grad(x, counts[:5], tokens, loss, 2),
              lambda: routing.balance_loss_grad(x, counts, tokens, loss.double(), 2),
              lambda: routing.balance_loss_grad(x, counts, tokens, loss, 2, out=torch.empty(8, 31, device=dev))):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: routing.balance_loss(torch.zeros(2, 1025, device=dev), torch.zeros(2, 1, dtype=torch.int32, device=dev)),
              lambda: routing.balance_loss_grad(x, counts, tokens, loss, 0)):
        with pytest.raises(ChimereError) as e:
            f()
        assert e.value.code == 1


# ------------------------------------------------------------ a routed layer, as used

def test_router_loss_and_experts_together(dev):
    """Router logits, choice, statistics and the experts in 8 bits, one after another on one stream, eagerly and as a graph:
    the loss and counts agree with the choice that the experts were given."""
    from chimere_amd import int8
    from test_gpu_int8 import close, experts_ref, layer_of
    T, E, K, H, F = 150, 32, 4, 256, 128
    layer = layer_of(E, F, H, 1, dev)
    g = torch.Generator(device="cuda").manual_seed(7)
    router, rs = int8.quantize_i8(torch.randn(E, H, generator=g, device=dev) * 0.05)
    x = torch.randn(T, H, generator=g, device=dev)
    ids, wts = torch.empty(T, K, dtype=torch.int32, device=dev), torch.empty(T, K, device=dev)
    logits, out = torch.empty(T, E, device=dev), torch.empty(T, H, device=dev)

    def step():
        int8.linear_i8(x, router, rs, out=logits)
        G.gpu_topk_softmax(logits, ids, wts, E, K, ntok=T)
        s = routing.balance_loss(logits, ids)
        grad = routing.balance_loss_grad(logits, s[1], s[3], s[0], K)
        layer.forward(x, ids, wts, out=out)
        return s, grad

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s, grad = step()
    for i in range(3):
        print(f"together replay {i}", flush=True)
        x.copy_(torch.randn(T, H, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert (ids.long().sort(1)[0] == logits.topk(K, dim=1)[1].sort(1)[0]).all()
        (rl, rc, rp, rn, rg), (tl, tp, tg) = ref(logits, ids, None, float(s[0]))
        assert (s[1].cpu() == rc).all() and int(s[3]) == T and abs(float(s[0]) - float(rl)) <= float(tl)
        assert ((s[2].double().cpu() - rp).abs() <= tp).all() and ((grad.double().cpu() - rg).abs() <= tg).all()
        close(out, *experts_ref(layer, x, ids, wts, torch.float32))


def test_far_logits(dev):
    """2.25 G logits, 2148 copies of 1024 rows: the loss, counts and probabilities of one copy, the gradient of each
    row that of the one copy.  Sums of equal terms differ by their roundings: at most 1024 in a row of a lane, 512 over
    waves and work-groups, on either side.  In a gradient c p (f - d), f has 3 roundings, d = sum f p those and at most
    22 of its own, on either side, the rest 10; both are rounded to bf16 (half a step each)."""
    copies, T, E, K = 2148, 1024, 1023, 4
    print("far logits", flush=True)
    x, ids, _ = choice(T, E, K, 3, torch.bfloat16, dev)
    one = torch.ones(1, device=dev)
    loss, counts, probs, tokens = routing.balance_loss(x, ids)
    grad = routing.balance_loss_grad(x, counts, tokens, one, K).double()
    big = x.repeat(copies, 1)
    bl, bc, bp, bt = routing.balance_loss(big, ids.repeat(copies, 1))
    bg = routing.balance_loss_grad(big, bc, bt, one * copies, K)
    assert int(bt) == copies * T and torch.equal(bc, counts * copies)
    tol = 2 * 1536 * U
    assert ((bp - probs).abs() <= tol * probs).all() and abs(float(bl) - float(loss)) <= 2 * tol * float(loss)
    p, f = torch.softmax(x.double(), 1), counts.double() / (T * K)
    tol = E / T * p * (6 * f + 50 * (p @ f)[:, None]) * U + 10 * U * grad.abs() + 2.02 * STEP[x.dtype] * grad.abs()
    for k in (0, copies // 2, copies - 1):
        assert ((bg[k * T:(k + 1) * T].double() - grad).abs() <= tol).all(), k
