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


@pytest.mark.parametrize("below", [28, 31, 33, 36, 40])
def test_chunk_of_small_weights(dev, below):
    """A chunk whose weights are each near or below the row's last bit (2^-46 of the largest at 32768 logits) and together are
    not: its tokens are drawn in proportion, and the logit before them, masked by the lowest number, never is.  All its weights
    are equal, so that a uniform number's token is known to the row's last bit: 16383 e^-below / (1 + 16383 e^-below) of the sum,
    rounded down to 2^-46, then the part of it that the number asks for."""
    V, n = 32768, 16383
    x = torch.full((1, V), -float("inf"), device=dev)
    x[0, 0] = torch.finfo(torch.float32).min
    x[0, 1:16384] = -float(below)
    x[0, 20000] = 0.0
    w = torch.exp(torch.tensor(-float(below), dtype=torch.float64)).item()
    part = n * w / (1 + n * w)
    u = torch.tensor([0.0, part * 0.001, part * 0.25, part * 0.5, part * 0.6, part * 1.01, 0.5, 1 - 2.0 ** -24], device=dev)
    token, logprob = sampling.sample(x.expand(8, V), u, **filled(8, dev))
    off = 2 + 2.0 ** -45 / w        # two tokens, and the last bit of the row's in tokens
    for i, (t, v) in enumerate(zip(token.tolist(), u.double().tolist())):
        if i < 5:
            assert 1 <= t < 16384 and abs(t - (1 + v * (1 + n * w) / w)) <= off, (i, t)
            assert abs(logprob[i].item() + below + n * w) < 2.0 ** -24 * below + 1e-9
        else:
            assert t == 20000, (i, t)
    assert token[0] == 1
    # a share that the largest has by itself leaves them out
    assert sampling.sample(x.expand(8, V), u, top_p=0.999999, **filled(8, dev))[0].tolist() == [20000] * 8


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [20000, 50257, 151936])
def test_chunks_of_all_heights(dev, V, dtype):
    """Chunks up to 45 octaves below the largest, uniform numbers down to 1e-14: the token is one with a weight, it is kept, and
    its share of the sum lies at the number, but for what sums are off by."""
    g = torch.Generator(device="cuda").manual_seed(V)
    n = 48
    x = torch.randn(n, V, generator=g, device=dev)
    for c in range(0, V, 16384):
        x[:, c:c + 16384] -= 31 * torch.rand(n, 1, generator=g, device=dev)
    x[torch.rand(n, V, generator=g, device=dev) < 0.3] = torch.finfo(TYPES[dtype]).min
    x[torch.rand(n, V, generator=g, device=dev) < 0.1] = -float("inf")
    x = x.to(TYPES[dtype])
    u = 10.0 ** (-14 * torch.rand(n, generator=g, device=dev))
    u[:3] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5], device=dev)
    wide = x.double().cpu()
    for t, p, m in ((1.0, 1.0, 0.0), (0.7, 1.0, 0.0), (1.0, 0.9999, 0.0), (1.3, 1.0, 1e-9), (1.0, 0.3, 0.5)):
        print(f"sample heights V={V} {dtype} T={t} top_p={p} min_p={m}", flush=True)
        token, logprob = sampling.sample(x, u, temperature=t, top_p=p, min_p=m, **filled(n, dev))
        t, p, m = (torch.tensor(v).item() for v in (t, p, m))
        w = torch.exp((wide - wide.max(1, keepdim=True)[0]) / t)
        down, order = torch.sort(w, dim=1, descending=True, stable=True)
        sums = torch.cumsum(down, 1)
        keep = (sums - down < p * sums[:, -1:] * (1 + 1e-7)) & (down >= m * (1 - 1e-7))
        kept = torch.zeros_like(keep).scatter(1, order, keep)
        at = token.cpu().long()
        rows = torch.arange(n)
        assert ((at >= 0) & (at < V)).all() and kept[rows, at].all() and (w[rows, at] > 0).all()
        w = torch.where(kept, w, torch.zeros_like(w))
        sums = torch.cumsum(w, 1)
        want = u.double().cpu() * sums[:, -1]
        off = 1e-6 * sums[:, -1] if p < 1 or m > 0 else (1e-12 + V * 2.0 ** -min(51, 62 - (V - 1).bit_length())) * sums[:, -1]
        past = sums[rows, at]
        assert (past >= want - off).all() and (past - w[rows, at] <= want + off).all()
        assert ((logprob.double().cpu() - torch.log(w[rows, at] / sums[:, -1])).abs() < 1e-5).all()


KINDS = ["power", "flat", "peak", "few", "grammar"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [1, 2, 3, 65, 1000, 1025, 4100, 20000, 50257, 151936])
def test_cuts_between_two_logits(dev, V, kind, dtype):
    """Shares, numbers and uniform numbers half way between two borders, so that every row is decided: the cut after any logit of
    more than 3e-7 of the sum (of thousands of equals too, by index), by each of the three ways and by all, and any token of such
    a weight.  A f32 in [0, 1) is off by 2^-25 = 3e-8, the sums by 1e-8 of themselves (V 2^-44), together less than half of the
    1.5e-7 to the next border."""
    g = torch.Generator(device="cuda").manual_seed(V + len(kind))
    h = torch.Generator().manual_seed(V)
    n = 8 if V < 20000 else 5
    x = logits(kind, n, V, g, dev).to(TYPES[dtype])
    wide = x.double().cpu()
    pick = lambda many: int(torch.randint(0, many, (1,), generator=h))  # noqa: E731
    for t in (1.0, 2.0):
        down, order = torch.sort(wide, dim=1, descending=True, stable=True)
        down = torch.exp((down - down[:, :1]) / t)
        for how in ("p", "k", "m", "kp", "all"):
            ks, ps, ms, us, want, logp = [], [], [], [], [], []
            for i in range(n):
                w, k, p, m = down[i], 0, 1.0, 0.0
                last = int((w > 0).sum())
                if how in ("k", "kp", "all"):
                    k = last = 1 + pick(min(last, 2500))
                total = float(w[:last].sum())
                if how in ("p", "kp", "all"):
                    last = 1 + pick(max(1, int((w[:last] > 3e-7 * total).sum())))
                    p = (float(w[:last].sum()) - float(w[last - 1]) / 2) / total
                if how in ("m", "all"):     # the last of a run of equals, well above the next
                    low = w[pick(last)]
                    next_ = w[w < low * (1 - 1e-5)]
                    m = float(torch.sqrt(low * next_[0])) if len(next_) and next_[0] > 0 else float(low) / 2
                    last = min(last, int((w >= m).sum()))
                    if ((w - m).abs() < 1e-6 * m).any():
                        m = 0.0
                        last = int((w > 0).sum()) if how == "m" else last
                kept = torch.sort(order[i, :last])[0]
                weight = torch.exp((wide[i, kept] - wide[i].max()) / t)
                total = float(weight.sum())
                heavy = torch.nonzero(weight > 3e-7 * total).view(-1)
                at = int(heavy[pick(len(heavy))])
                ks.append(k), ps.append(p), ms.append(m)
                us.append((float(weight[:at].sum()) + float(weight[at]) / 2) / total)
                want.append(int(kept[at]))
                logp.append(float(torch.log(weight[at] / total)))
            if how == "all" and 0.0 in ms:      # (the share's cut was found with min_p's)
                continue
            print(f"sample between V={V} {kind} {dtype} T={t} by {how} k={ks} p={ps} m={ms}", flush=True)
            f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
            token, logprob = sampling.sample(x, f32(us), temperature=t, top_k=torch.tensor(ks, dtype=torch.int32, device=dev), top_p=f32(ps), min_p=f32(ms), **filled(n, dev))
            assert token.tolist() == want, (token.tolist(), want, us)
            off = torch.tensor(logp, dtype=torch.float64)
            assert ((logprob.double().cpu() - off).abs() <= 2.0 ** -24 * off.abs() + 3e-8).all()
