"""The 8-bit integer products and the router's balance loss, as a server and a trainer of a routed-MoE model call them.

Three kinds of call:

* ``linear``: float tokens against a matrix of 8-bit integers with one scale per output channel; the tokens are quantized
  within the call, one scale each;
* ``experts``: the routed experts' FFN in the same format, for tokens whose expert ids and weights the router has given;
* ``balance``: per-expert counts and the balance loss of a router's choice, and the gradient of its logits.

Layer shapes are the benchmark's (hidden 2048, 256 experts of 512, top-8) and sizes around them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
WEIGHT_STD = 0.02       # trained projections are near N(0, 0.02)


def listed():
    moe = {"kind": "experts", "H": 2048, "F": 512, "E": 256, "K": 8}
    return [
        # a decode token's small projection: latency
        {"name": "linear_1_4096x2048", "kind": "linear", "M": 1, "N": 4096, "C": 2048, "x": "bf16", "out": "bf16", "bias": False},
        # the output head of a decode batch, logits in 32 bits
        {"name": "linear_8_151936x2048", "kind": "linear", "M": 8, "N": 151936, "C": 2048, "x": "f32", "out": "f32", "bias": False},
        # a short prompt of odd length through a projection with a bias
        {"name": "linear_77_2048x4096", "kind": "linear", "M": 77, "N": 2048, "C": 4096, "x": "f16", "out": "f16", "bias": True},
        # the usual prompt chunk through a wide projection
        {"name": "linear_512_8192x2048", "kind": "linear", "M": 512, "N": 8192, "C": 2048, "x": "bf16", "out": "bf16", "bias": False},
        # a long prompt's chunk, the largest product
        {"name": "linear_4096_8192x4096", "kind": "linear", "M": 4096, "N": 8192, "C": 4096, "x": "f32", "out": "bf16", "bias": False},
        # one decode token through its experts
        dict(moe, name="experts_1", T=1, x="bf16", out="bf16"),
        # a short prompt
        dict(moe, name="experts_45", T=45, x="f32", out="f16"),
        # the usual prompt chunk
        dict(moe, name="experts_512", T=512, x="bf16", out="bf16"),
        # a long prompt's chunk
        dict(moe, name="experts_4096", T=4096, x="bf16", out="bf16"),
        # the router's statistics of one small step
        {"name": "balance_64", "kind": "balance", "T": 64, "E": 256, "K": 8, "x": "f32", "pad": 0.0, "drop": 0.0},
        # a padded batch with pairs dropped for capacity
        {"name": "balance_4099", "kind": "balance", "T": 4099, "E": 256, "K": 8, "x": "bf16", "pad": 0.2, "drop": 0.05},
        # a training step's tokens
        {"name": "balance_32768", "kind": "balance", "T": 32768, "E": 256, "K": 8, "x": "f32", "pad": 0.1, "drop": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "experts", "balance"])
    types = ["f32", "f16", "bf16"]
    if kind == "linear":
        # tokens: one, a decode batch, a chunk; no more than the largest listed product, output and matrix
        m = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 4096), _log(rng, 17, 4096)])
        c = _log(rng, 128, 8192)
        c = c if rng.random() < 0.3 else max(64, c // 64 * 64)
        n = _log(rng, 64, min(151936, 300_000_000 // c, 2 ** 37 // (m * c)))
        x = rng.choice(types)
        return {"kind": kind, "M": m, "N": n, "C": c, "x": x, "out": rng.choice([x, "f32", "bf16"]), "bias": rng.random() < 0.3}
    if kind == "experts":
        h, f = 64 * _log(rng, 4, 64), 64 * _log(rng, 2, 32)
        e = rng.choice([8, 16, 60, 64, 128, 256])
        e = max(8, min(e, 900_000_000 // (3 * h * f)))
        k = rng.randint(1, 8)
        t = rng.choice([rng.randint(1, 8), _log(rng, 9, 4096), _log(rng, 9, 4096)])
        t = max(1, min(t, 4096 * 8 * 2048 * 512 // (k * h * f)))
        x = rng.choice(types)
        return {"kind": kind, "H": h, "F": f, "E": e, "K": k, "T": t, "x": x, "out": "f16" if x == "f16" else "bf16"}
    e = _log(rng, 8, 1024)
    return {"kind": kind, "T": _log(rng, 1, min(32768, 32768 * 256 // e)), "E": e, "K": rng.randint(1, min(e, 10)), "x": rng.choice(types),
            "pad": rng.choice([0.0, rng.random()]), "drop": rng.choice([0.0, 0.3 * rng.random()])}


# ------------------------------------------------------------ inputs

def _weights(shape, g, dev):
    """Weights in 8 bits, rows 16-byte aligned, and the scale of each row."""
    rows, c = shape[:-1], shape[-1]
    q = torch.zeros(*rows, (c + 15) // 16 * 16, dtype=torch.int8, device=dev)
    scale = torch.empty(rows, device=dev)
    lead = q.view(-1, q.shape[-1])
    step = max(1, (1 << 27) // c)
    for r in range(0, lead.shape[0], step):
        w = torch.randn(min(step, lead.shape[0] - r), c, generator=g, device=dev) * WEIGHT_STD
        s = w.abs().amax(1) / 127
        lead[r:r + step, :c] = (w / s[:, None]).round().to(torch.int8)
        scale.view(-1)[r:r + step] = s
    return q[..., :c], scale


def _tokens(n, c, dtype, g, dev):
    """Activations: some channels larger than others, as a trained model's are."""
    channel = torch.exp(0.5 * torch.randn(c, generator=g, device=dev))
    return (torch.randn(n, c, generator=g, device=dev) * channel).to(DTYPES[dtype])


def _logits(n, e, dtype, g, dev):
    """Router logits with favoured experts."""
    return (1.5 * torch.randn(n, e, generator=g, device=dev) + 0.5 * torch.randn(e, generator=g, device=dev)).to(DTYPES[dtype])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "linear":
        s["x"] = _tokens(case["M"], case["C"], case["x"], g, dev)
        s["w"], s["w_scale"] = _weights((case["N"], case["C"]), g, dev)
        s["bias"] = torch.randn(case["N"], generator=g, device=dev) if case["bias"] else None
        s["out"] = torch.empty(case["M"], case["N"], dtype=DTYPES[case["out"]], device=dev)
        return s
    e, k, t = case["E"], case["K"], case["T"]
    logits = _logits(t, e, case["x"] if case["kind"] == "balance" else "f32", g, dev)
    p, ids = torch.softmax(logits.float(), 1).topk(k, dim=1)
    s["ids"] = ids.to(torch.int32)
    if case["kind"] == "experts":
        h, f = case["H"], case["F"]
        s["wts"] = p / p.sum(1, keepdim=True)
        s["x"] = _tokens(t, h, case["x"], g, dev)
        for name, shape in (("gate", (e, f, h)), ("up", (e, f, h)), ("down", (e, h, f))):
            s[name], s[name + "_scale"] = _weights(shape, g, dev)
        s["out"] = torch.empty(t, h, dtype=DTYPES[case["out"]], device=dev)
        return s
    s["logits"] = logits
    s["ids"][torch.rand(t, k, generator=g, device=dev) < case["drop"]] = -1
    s["mask"] = torch.rand(t, generator=g, device=dev) >= case["pad"] if case["pad"] else None
    s["grad_loss"] = torch.full((1,), 0.01, device=dev)
    s["grad"] = torch.empty_like(logits)
    return s


# ------------------------------------------------------------ the plain forms

def _quantize(x):
    scale = x.abs().amax(-1, keepdim=True) / 127
    return torch.where(scale > 0, x / scale, torch.zeros_like(x)).round(), scale


def _linear(s):
    q, scale = _quantize(s["x"].float())
    y = q @ s["w"].float().T * scale * s["w_scale"]
    return y if s["bias"] is None else y + s["bias"]


def _ffn(x, s, pick):
    """Batches x [n, rows, H] through the experts that `pick` takes, a batch each."""
    q, scale = _quantize(x)
    g, u = (torch.bmm(q, s[w][pick].float().transpose(1, 2)) * scale * s[w + "_scale"][pick][:, None] for w in ("gate", "up"))
    q, scale = _quantize(g / (1 + torch.exp(-g)) * u)
    return torch.bmm(q, s["down"][pick].float().transpose(1, 2)) * scale * s["down_scale"][pick][:, None]


def _experts(s):
    c, x = s["case"], s["x"].float()
    t, k, e = c["T"], c["K"], c["E"]
    ids = s["ids"].reshape(-1).long()
    rows = torch.arange(t * k, device=x.device) // k
    if t * k <= 64:     # a few pairs: each with its expert's weights
        y = _ffn(x[rows][:, None], s, ids)[:, 0]
    else:               # the pairs of each expert as one batch, filled up to the longest
        order = torch.argsort(ids, stable=True)
        count = torch.zeros(e, dtype=torch.long, device=x.device).index_add_(0, ids, torch.ones_like(ids))
        slot = torch.arange(t * k, device=x.device) - (torch.cumsum(count, 0) - count)[ids[order]]
        batch = torch.zeros(e, int(count.max()), c["H"], device=x.device)
        batch[ids[order], slot] = x[rows[order]]
        y = torch.empty(t * k, c["H"], device=x.device)
        y[order] = _ffn(batch, s, slice(None))[ids[order], slot]
    return (y.view(t, k, -1) * s["wts"][..., None]).sum(1)


def _balance(s):
    c = s["case"]
    e, k = c["E"], c["K"]
    logits = s["logits"].float()
    keep = torch.ones(c["T"], dtype=torch.bool, device=logits.device) if s["mask"] is None else s["mask"]
    n = keep.sum()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    p = torch.where(keep[:, None], p, torch.zeros_like(p))
    ids = torch.where(keep[:, None] & (s["ids"] >= 0), s["ids"], torch.full_like(s["ids"], e)).reshape(-1).long()
    counts = torch.zeros(e + 1, dtype=torch.int32, device=logits.device).index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))[:e]
    some = n.clamp_min(1).float()
    share, mean = counts / (some * k), p.sum(0) / some
    loss = e * (share * mean).sum()
    grad = s["grad_loss"] * (e / some) * p * (share - (p * share).sum(1, keepdim=True))
    return {"loss": loss.view(1), "counts": counts, "probs": mean, "grad": grad.to(s["logits"].dtype)}


# ------------------------------------------------------------ the calls

def run(s):
    c = s["case"]
    if own:
        if c["kind"] == "linear":
            from chimere_amd import int8
            return int8.linear_i8(s["x"], s["w"], s["w_scale"], bias=s["bias"], out=s["out"])
        if c["kind"] == "experts":
            from chimere_amd import int8
            if "layer" not in s:    # the handle that a program makes once, next to its weights
                s["layer"] = int8.Int8Experts(*(s[n + t] for n in ("gate", "up", "down") for t in ("", "_scale")))
            return s["layer"].forward(s["x"], s["ids"], s["wts"], out=s["out"])
        from chimere_amd import routing
        loss, counts, probs, tokens = routing.balance_loss(s["logits"], s["ids"], mask=s["mask"])
        grad = routing.balance_loss_grad(s["logits"], counts, tokens, s["grad_loss"], c["K"], mask=s["mask"], out=s["grad"])
        return {"loss": loss, "counts": counts, "probs": probs, "grad": grad}
    if c["kind"] == "balance":
        return _balance(s)
    return (_linear(s) if c["kind"] == "linear" else _experts(s)).to(DTYPES[c["out"]])


def work(case):
    if case["kind"] == "linear":
        m, n, c = case["M"], case["N"], case["C"]
        return {"bytes": m * c * SIZE[case["x"]] + n * c + 4 * n * (2 if case["bias"] else 1) + m * n * SIZE[case["out"]], "flops": 2 * m * n * c}
    e, k, t = case["E"], case["K"], case["T"]
    if case["kind"] == "experts":
        h, f = case["H"], case["F"]
        distinct = e * (1 - (1 - k / e) ** t)        # experts that t tokens' routing meets
        return {"bytes": int(distinct * (3 * h * f + 8 * f + 4 * h)) + t * h * (SIZE[case["x"]] + SIZE[case["out"]]) + 8 * t * k,
                "flops": 6 * t * k * h * f}
    kept = t * (1 - case["pad"])
    return {"bytes": int(kept * (e * SIZE[case["x"]] + 4 * k)) + t * e * SIZE[case["x"]] + t + 8 * e, "flops": 12 * kept * e}


# ------------------------------------------------------------ in 64 bits

def _q64(x):
    """The integers of a row and its scale: the scale and the quotients are 32-bit numbers by definition."""
    scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
    q = torch.round((x / torch.where(scale > 0, scale, torch.ones_like(scale))).float().double())
    return q, scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        q, scale = _q64(s["x"].double())
        y = torch.cat([q @ w.double().T for w in s["w"].split(16384)], 1) * scale * s["w_scale"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "experts":
        x = s["x"].double()
        y = torch.zeros_like(x)
        for e in range(case["E"]):
            t, k = torch.nonzero(s["ids"] == e, as_tuple=True)
            if t.numel():
                q, scale = _q64(x[t])
                g = q @ s["gate"][e].double().T * scale * s["gate_scale"][e].double()
                u = q @ s["up"][e].double().T * scale * s["up_scale"][e].double()
                q, scale = _q64(g * torch.sigmoid(g) * u)
                y.index_add_(0, t, s["wts"][t, k, None].double() * (q @ s["down"][e].double().T * scale * s["down_scale"][e].double()))
        return y
    e, k = case["E"], case["K"]
    keep = torch.ones(case["T"], dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    n = max(float(keep.sum()), 1.0)
    p = torch.softmax(s["logits"].double(), 1) * keep[:, None]
    here = s["ids"][keep > 0].reshape(-1)
    f = torch.bincount(here[here >= 0], minlength=e).double() / (n * k)
    loss = e * (f @ p.sum(0)) / n
    grad = float(s["grad_loss"]) * e / n * p * (f - (p @ f)[:, None])
    return {"loss": loss.view(1), "counts": None, "probs": p.sum(0) / n, "grad": grad}
