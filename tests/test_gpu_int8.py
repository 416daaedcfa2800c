"""Products over 8-bit integers (quantize_i8, gemm_i8, linear_i8, Int8Experts)
against plain 64-bit forms.

Tolerances, per element, u = 2^-24 (half a step of f32):
* integers and scales of the quantizer: equal (defined by one f32 product and
  f32 quotients, which numpy rounds alike);
* a product: the int32 sum is exact; its conversion and the two scalings round
  once each (3 u of the product), the bias once (u of the result), and the
  result once more to the output type (eps / 2);
* the experts: h carries a relative error of at most 16 u (two products of 3 u,
  an exponential of 2 u whose argument's error 3 u |g| is largest where
  silu(g) is smallest, bounded with g's own size; a division, two products).
  An integer of h may then be one step off where its quotient lies within that
  error of a half: each such place adds its step times |D|."""
import numpy as np
import pytest
import torch

from chimere_amd import int8
from chimere_amd._lib import ChimereError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def q_ref(x):
    """The quantizer's definition in numpy: x float32 [n, c] -> (integers float64, scale float64)."""
    x = x.detach().float().cpu().numpy()
    bits = (x.view(np.uint32) & 0x7FFFFFFF).max(1)
    with np.errstate(all="ignore"):
        scale = bits.view(np.float32) * (np.float32(1) / np.float32(127))
        q = np.rint(x / scale[:, None]).clip(-127, 127)
    q[~((scale > 0) & np.isfinite(scale))] = 0
    return torch.from_numpy(q.astype(np.float64)), torch.from_numpy(scale.astype(np.float64))


def weights(n, c, g, pad=0):
    """int8 rows with garbage behind them, and scales."""
    w = torch.randint(-128, 128, (n, (c + 15) // 16 * 16 + pad), generator=g, device="cuda", dtype=torch.int8)
    return w[:, :c], torch.rand(n, generator=g, device="cuda") * 1e-3 + 1e-4


def close(out, ref, tol):
    bad = (out.double().cpu() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), (out.double().cpu() - ref)[bad][:4], tol[bad][:4], ref[bad][:4])


def product(q, s, w, ws, bias, dtype):
    """(reference, tolerance) of a product of integers q (float64) with scales s."""
    y = (q @ w.double().cpu().T) * s[:, None] * ws.double().cpu()
    tol = 3.01 * U * y.abs()
    if bias is not None:
        y = y + bias.double().cpu()
        tol = tol + U * y.abs()
    return y, tol * (1 + STEP[dtype]) + STEP[dtype] * y.abs() + TINY[dtype]


# ------------------------------------------------------------ quantizer

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (1, 2048), (3, 7), (5, 16), (2, 1000), (7, 2047), (4, 4096), (3, 8192), (2, 8200),
                                 (2, 20001), (300, 256)])
def test_quantize(dev, n, c, dtype):
    print(f"quantize {n}x{c} {dtype}", flush=True)
    x = (torch.randn(n, c, generator=gen(n * c), device=dev) * 3).to(TYPES[dtype])
    q, s = int8.quantize_i8(x)
    rq, rs = q_ref(x)
    assert (s.double().cpu() == rs).all()
    assert (q.double().cpu() == rq).all()


@pytest.mark.parametrize("c", [64, 100, 2048, 9000])
def test_quantize_borders(dev, c):
    """Quotients at and next to halves, subnormal and huge rows, zeros, infinities and NaN."""
    print(f"quantize borders {c}", flush=True)
    g = gen(c)
    half = torch.randint(-127, 127, (1, c), generator=g, device=dev).float() + 0.5
    half[0, 0] = 127.0
    rows = [half, half * 3, half / 7, half * 2.0 ** -149, half * 2.0 ** -140, half * 2.0 ** -120, half * 2.0 ** 120,
            torch.nextafter(half, torch.zeros_like(half)), torch.nextafter(half * 0.37, half * 1e3),
            half * 1.5 * 2.0 ** -149, half * 2.3 * 2.0 ** -149, torch.zeros(1, c, device=dev), -torch.zeros(1, c, device=dev)]
    x = torch.cat(rows)
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = torch.randn(1, c, generator=g, device=dev)
        r[0, c - 1] = bad
        x = torch.cat([x, r])
    q, s = int8.quantize_i8(x)
    rq, rs = q_ref(x)
    assert ((s.double().cpu() == rs) | (s.double().cpu().isnan() & rs.isnan())).all()
    assert (q.double().cpu() == rq).all()


def test_quantize_many_short_rows(dev):
    """More rows than one grid of a wave each has threads for: a single element is its own maximum."""
    n = (1 << 26) + 5
    x = torch.randint(-3, 4, (n, 1), generator=gen(5), device=dev).to(torch.bfloat16)
    q, s = int8.quantize_i8(x)
    assert (q == torch.sign(x).to(torch.int8) * 127).all()
    assert (s == x.abs().float().flatten() * torch.full((1,), 1.0 / 127, device=dev)).all()


@pytest.mark.parametrize("power", [-140, -100, -89, -20, 0, 60, 115])
def test_quantize_next_to_ties(dev, power):
    """16 million quotients within two steps of a half, for 1024 scales of every mantissa length."""
    g = gen(power + 200)
    amax = (torch.rand(1024, 1, generator=g, device=dev) + 1) * 127.0
    amax[::3] = torch.floor(amax[::3] * 64) / 64
    amax = (amax.double() * 2.0 ** power).float()
    scale = amax * torch.full((1,), 1.0 / 127, device=dev)
    half = torch.randint(-127, 127, (1024, 16384), generator=g, device=dev) + 0.5
    x = (half.double() * scale.double()).float()
    for _ in range(2):
        way = torch.randint(0, 3, x.shape, generator=g, device=dev)
        x = torch.where(way == 0, torch.nextafter(x, -amax), torch.where(way == 1, torch.nextafter(x, amax), x))
    x[:, :1] = amax
    q, s = int8.quantize_i8(x)
    rq, rs = q_ref(x)
    assert (s.double().cpu() == rs).all() and (q.double().cpu() == rq).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_quantize_many_ties(dev, dtype):
    """Rows whose largest value is a multiple of 127 in its last places, so that every other one is a tie; scales as torch's."""
    g = gen(1)
    x = torch.randint(-254, 255, (200, 300), generator=g, device=dev)
    x[:, 0] = 254
    x = (x.float() * 2.0 ** torch.randint(-8, 5, (200, 1), generator=g, device=dev)).to(TYPES[dtype])
    q, s = int8.quantize_i8(x)
    rq, rs = q_ref(x)
    assert (s.double().cpu() == rs).all() and (q.double().cpu() == rq).all()
    assert (s == x.float().abs().amax(1) / 127).all()


def test_quantize_strides_and_what_is_left(dev):
    """Rows apart in x (also on odd addresses) and q; what lies between q's rows stays."""
    for c, off, dtype in ((100, 3, torch.float32), (100, 1, torch.bfloat16), (2048, 0, torch.float16), (33, 5, torch.float16)):
        print(f"quantize strides {c} {off} {dtype}", flush=True)
        x = torch.randn(6, c + 37, generator=gen(c), device=dev).to(dtype)[:, off:off + c]
        room = torch.full((6, (c + 15) // 16 * 16 + 32), 77, dtype=torch.int8, device=dev)
        q, s = int8.quantize_i8(x, q=room[:, :c])
        rq, rs = q_ref(x)
        assert (q.double().cpu() == rq).all() and (s.double().cpu() == rs).all()
        assert (room[:, c:] == 77).all()
    x = torch.randn(1, 256, device=dev).expand(4, 256)                  # one row read four times
    q, s = int8.quantize_i8(x)
    assert (q == q[:1]).all() and (q.double().cpu() == q_ref(x)[0]).all()


# ------------------------------------------------------------ dense product

SHAPES = [(1, 1, 1), (1, 4096, 2048), (1, 17, 100), (2, 300, 4100), (3, 65, 17), (4, 2000, 512), (5, 129, 15), (8, 1000, 2048),
          (9, 333, 257), (16, 515, 1024), (17, 64, 128), (31, 40, 96), (33, 130, 129), (45, 2048, 640), (64, 64, 64),
          (65, 257, 1000), (77, 512, 4096), (100, 1030, 333), (128, 128, 256), (130, 700, 383), (200, 3000, 512),
          (257, 260, 1025), (300, 1537, 130), (513, 1000, 700), (700, 4100, 258), (1030, 2050, 384), (2100, 1100, 200)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,c", SHAPES)
def test_gemm(dev, m, n, c, dtype):
    print(f"gemm {m}x{n}x{c} {dtype}", flush=True)
    g = gen(m * 7 + n * 3 + c)
    a, s = weights(m, c, g)
    w, ws = weights(n, c, g, pad=16)
    bias = torch.randn(n, generator=g, device=dev) if (m + n) % 2 else None
    out = int8.gemm_i8(a, s, w, ws, bias=bias, dtype=TYPES[dtype])
    close(out, *product(a.double().cpu(), s.double().cpu(), w, ws, bias, TYPES[dtype]))


@pytest.mark.parametrize("m", [1, 2, 20, 150, 600])
def test_gemm_longest_rows_of_extremes(dev, m):
    """131071 columns of -128 and 127: the largest sums that int32 holds."""
    print(f"gemm extremes {m}", flush=True)
    c, n = 131071, 40
    a = torch.full((m, 131072), -128, dtype=torch.int8, device=dev)[:, :c]
    w = torch.full((n, 131072), -128, dtype=torch.int8, device=dev)[:, :c]
    w[1::2] = 127
    one_m, one_n = torch.ones(m, device=dev), torch.ones(n, device=dev)
    out = int8.gemm_i8(a, one_m, w, one_n)
    ref = torch.where(torch.arange(n) % 2 == 0, 128.0 * 128 * c, -128.0 * 127 * c).double().expand(m, n)
    close(out, ref, U * ref.abs())


@pytest.mark.parametrize("m,n,c", [(1, 100, 64), (7, 200, 100), (70, 90, 300), (300, 600, 200)])
def test_gemm_strides_and_what_is_left(dev, m, n, c):
    """Rows apart on all sides, an output on an odd address; what lies around the output stays."""
    print(f"gemm strides {m} {n} {c}", flush=True)
    for dtype in TYPES.values():
        g = gen(n)
        a, s = weights(m, c, g, pad=48)
        w, ws = weights(n, c, g, pad=112)
        room = torch.full((m + 2, n + 11), 5.0, dtype=dtype, device=dev)
        int8.gemm_i8(a, s, w, ws, out=room[1:m + 1, 3:n + 3])
        close(room[1:m + 1, 3:n + 3], *product(a.double().cpu(), s.double().cpu(), w, ws, None, dtype))
        room[1:m + 1, 3:n + 3] = 5.0
        assert (room == 5.0).all()


@pytest.mark.parametrize("xt", TYPES)
@pytest.mark.parametrize("m,n,c", [(1, 4096, 2048), (1, 5, 1), (1, 1000, 4097), (2, 70, 300), (3, 1000, 2048), (8, 513, 1024), (12, 100, 9000), (4, 8192, 2048), (4, 500, 2049), (3, 8200, 512), (2, 9001, 4000), (1, 8193, 8192), (1, 40, 8193),
                                   (40, 300, 500), (300, 500, 129), (16, 2048, 512), (17, 700, 480), (64, 2048, 512), (100, 90, 512),
                                   (500, 200, 256), (513, 250, 100), (8, 300, 2048), (16, 1000, 1000), (40, 513, 1024), (33, 100, 1025),
                                   (8, 16384, 512), (5, 16400, 500), (5, 1, 3000), (1000, 1, 16), (2, 8192, 8192)])
def test_linear(dev, m, n, c, xt):
    print(f"linear {m}x{n}x{c} {xt}", flush=True)
    g = gen(m + n + c)
    x = torch.randn(m, c, generator=g, device=dev).to(TYPES[xt])
    w, ws = weights(n, c, g)
    q, s = q_ref(x)
    for dtype in TYPES.values():
        close(int8.linear_i8(x, w, ws, dtype=dtype), *product(q, s, w, ws, None, dtype))
    room = torch.randn(m, c + 9, generator=g, device=dev).to(TYPES[xt])[:, 5:5 + c]     # odd addresses
    q, s = q_ref(room)
    bias = torch.randn(n, generator=g, device=dev)
    out = int8.linear_i8(room, w, ws, bias=bias)
    close(out, *product(q, s, w, ws, bias, TYPES[xt]))
    qd, sd = int8.quantize_i8(room)
    assert (int8.gemm_i8(qd, sd, w, ws, bias=bias, dtype=out.dtype) == out).all()       # the same, in two calls


def test_linear_rows_do_not_depend_on_each_other(dev):
    """A token's row has the same bits alone, in a decode batch and in a chunk; a NaN stays in its row."""
    g = gen(5)
    x = torch.randn(600, 1000, generator=g, device=dev)
    x[3, 17] = float("nan")
    x[4, 0] = float("inf")
    x[5] = 0
    w, ws = weights(2050, 1000, g)
    full = int8.linear_i8(x, w, ws)
    assert full[3:5].isnan().all() and (full[5] == 0).all()
    for m in (1, 2, 3, 7, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 257, 400):
        print(f"linear rows {m}", flush=True)
        part = int8.linear_i8(x[:m], w, ws)
        same = (part == full[:m]) | (part.isnan() & full[:m].isnan())
        assert same.all(), m
    w = w[:300]
    for m in range(1, 120, 7):          # few work-groups: quantized by each
        part = int8.linear_i8(x[:m], w, ws[:300])
        same = (part == full[:m, :300]) | (part.isnan() & full[:m, :300].isnan())
        assert same.all(), m


def test_no_tokens(dev):
    w, ws = weights(30, 64, gen(1))
    assert int8.linear_i8(torch.empty(0, 64, device=dev), w, ws).shape == (0, 30)
    q, s = int8.quantize_i8(torch.empty(0, 64, device=dev))
    assert int8.gemm_i8(q, s, w, ws).shape == (0, 30)


# ------------------------------------------------------------ the experts

def layer_of(E, F, H, seed, dev):
    g = gen(seed)
    return int8.Int8Experts.from_float(*(torch.randn(E, r, c, generator=g, device=dev) * 0.05
                                         for r, c in ((F, H), (F, H), (H, F))))


def experts_ref(layer, x, ids, wts, dtype):
    gate, gs, up, us, down, ds = (t.double().cpu() for t in layer.tensors)
    T, K = ids.shape
    ids, wts = ids.cpu().long(), wts.double().cpu()
    xq, xs = q_ref(x)
    out, tol = torch.zeros(T, layer.H, dtype=torch.float64), torch.zeros(T, layer.H, dtype=torch.float64)
    for e in range(layer.E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        gg = xq[t] @ gate[e].T * xs[t, None] * gs[e]
        uu = xq[t] @ up[e].T * xs[t, None] * us[e]
        h = gg / (1 + torch.exp(-gg)) * uu
        rel = (16 + 3 * gg.abs()) * U                        # of h
        amax, where = h.abs().max(1, keepdim=True)
        srel = rel.gather(1, where) + 2 * U + (rel * h.abs()).amax(1, keepdim=True) / amax.clamp_min(1e-300)
        s = amax / 127
        quot = torch.where(s > 0, h / s.clamp_min(1e-300), torch.zeros_like(h))
        hq = torch.round(quot)
        err = quot.abs() * (rel + srel)
        near = ((quot - torch.floor(quot) - 0.5).abs() <= err).double()
        y = hq @ down[e].T * s * ds[e]
        ey = y.abs() * (srel + 4 * U) + near @ down[e].abs().T * s * ds[e]
        w = wts[t, k, None]
        out.index_add_(0, t, w * y)
        # for 16-bit outputs a pair's sum is held as f16: half a step, 2^-11 of it
        half = 0.0 if dtype == torch.float32 else 2.0 ** -11
        tol.index_add_(0, t, w.abs() * (ey + (y.abs() + ey) * ((K + 2) * U + half)))
    return out, tol * (1 + STEP[dtype]) + STEP[dtype] * out.abs() + TINY[dtype]


def routed(T, E, K, g, dev):
    p, ids = torch.softmax(torch.randn(T, E, generator=g, device=dev), 1).topk(K, dim=1)
    return ids.to(torch.int32), p / p.sum(1, keepdim=True)


@pytest.mark.parametrize("T,E,K,H,F", [(1, 4, 1, 16, 16), (1, 32, 8, 1024, 256), (2, 8, 3, 320, 48), (5, 16, 4, 256, 512),
                                       (8, 64, 8, 512, 128), (9, 8, 2, 128, 1040), (33, 3, 2, 144, 80), (40, 64, 8, 256, 192),
                                       (200, 8, 4, 272, 320), (300, 2, 1, 128, 64), (500, 40, 6, 512, 256), (700, 16, 16, 192, 512),
                                       (1500, 5, 2, 256, 704), (90, 40, 8, 256, 192), (300, 100, 3, 320, 208), (130, 50, 4, 144, 80),
                                       (1030, 1000, 2, 64, 32), (600, 8, 1, 1040, 272), (200, 30, 3, 160, 1040), (20, 2, 2, 4096, 2048),
                                       (1, 16, 8, 384, 1152), (2, 16, 8, 256, 2048), (1, 16, 8, 256, 4096), (3, 12, 4, 272, 4112), (1, 40, 16, 144, 1024),
                                       (1, 20, 16, 128, 2048), (1, 9, 1, 4096, 8192)])
def test_experts(dev, T, E, K, H, F):
    g = gen(T + E)
    layer = layer_of(E, F, H, T * E, dev)
    ids, wts = routed(T, E, K, g, dev)
    for xt, dtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)):
        print(f"experts T={T} E={E} K={K} H={H} F={F} {xt} {dtype}", flush=True)
        x = torch.randn(T, H, generator=g, device=dev).to(xt)
        close(layer.forward(x, ids, wts, dtype=dtype), *experts_ref(layer, x, ids, wts, dtype))


@pytest.mark.parametrize("T,E", [(1, 12), (6, 12), (90, 12), (400, 12), (150, 40)])
def test_experts_odd_choices(dev, T, E):
    """Ids that are no expert, the same expert twice, one expert for all, a token without any, strided rows, NaN."""
    K, H, F = 4, 256, 128
    layer = layer_of(E, F, H, 9, dev)
    g = gen(T)
    x = torch.randn(T, H + 24, generator=g, device=dev)[:, 7:7 + H]
    wts = torch.randn(T, K, generator=g, device=dev)
    choices = [torch.randint(-3, E + 3, (T, K), generator=g, device=dev), torch.full((T, K), 5, device=dev),
               torch.full((T, K), -1, device=dev), torch.tensor([2**31 - 1, -2**31, E, 0], device=dev).expand(T, K)]
    for i, ids in enumerate(choices):
        print(f"experts odd T={T} choice {i}", flush=True)
        ids = ids.to(torch.int32).contiguous()
        room = torch.full((T, H + 10), 3.0, device=dev)
        layer.forward(x, ids, wts, out=room[:, 1:H + 1])
        close(room[:, 1:H + 1], *experts_ref(layer, x, ids, wts, torch.float32))
        assert (room[:, 0] == 3.0).all() and (room[:, H + 1:] == 3.0).all()
    x = x.clone()
    x[0, 3] = float("nan")
    ids = torch.randint(0, E, (T, K), generator=g, device=dev).to(torch.int32)
    out = layer.forward(x, ids, wts)
    assert out[0].isnan().all() and not out[1:].isnan().any()


def test_experts_rows_do_not_depend_on_each_other(dev):
    E, K, H, F = 24, 6, 320, 208
    layer, g = layer_of(E, F, H, 3, dev), gen(4)
    x = torch.randn(700, H, generator=g, device=dev)
    ids, wts = routed(700, E, K, g, dev)
    full = layer.forward(x, ids, wts)
    for m in (1, 2, 3, 7, 8, 9, 16, 40, 90, 100, 333):
        print(f"experts rows {m}", flush=True)
        assert (layer.forward(x[:m], ids[:m].contiguous(), wts[:m].contiguous()) == full[:m]).all(), m
    assert layer.forward(x[:0], ids[:0].contiguous(), wts[:0].contiguous()).shape == (0, H)


# ------------------------------------------------------------ streams, graphs, refusals

def test_graph_replays_and_other_streams(dev):
    """Captured calls replayed on new inputs, with eager calls between; calls on two streams at once."""
    E, K, H, F = 16, 4, 256, 128
    layer, g = layer_of(E, F, H, 2, dev), gen(8)
    w, ws = weights(700, H, g)
    for T in (1, 5, 150):
        x, (ids, wts) = torch.randn(T, H, generator=g, device=dev), routed(T, E, K, g, dev)
        out, y = torch.empty(T, H, device=dev), torch.empty(T, 700, device=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.forward(x, ids, wts, out=out)
            int8.linear_i8(x, w, ws, out=y)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.forward(x, ids, wts, out=out)
            int8.linear_i8(x, w, ws, out=y)
        for i in range(4):
            print(f"graph T={T} replay {i}", flush=True)
            x.copy_(torch.randn(T, H, generator=g, device=dev))
            new_ids, new_w = routed(T, E, K, g, dev)
            ids.copy_(new_ids)
            wts.copy_(new_w)
            graph.replay()
            with torch.cuda.stream(side):
                other = layer.forward(x * 0 + 1, ids * 0, wts)      # beside the replay
            want, want_y = layer.forward(x, ids, wts), int8.linear_i8(x, w, ws)
            torch.cuda.synchronize()
            assert (out == want).all() and (y == want_y).all() and other.isfinite().all()


def test_refusals(dev):
    w, ws = weights(32, 64, gen(1))
    x = torch.randn(4, 64, device=dev)
    q, s = int8.quantize_i8(x)
    bad = [lambda: int8.linear_i8(x.double(), w, ws), lambda: int8.linear_i8(x[:, :32], w, ws),
           lambda: int8.linear_i8(x.t(), w, ws), lambda: int8.linear_i8(x, w, ws[:5]),
           lambda: int8.linear_i8(x, w, ws.double()), lambda: int8.linear_i8(x, w.float(), ws),
           lambda: int8.linear_i8(x, w, ws, bias=ws[:3]), lambda: int8.linear_i8(x.cpu(), w, ws),
           lambda: int8.linear_i8(x, w.cpu(), ws), lambda: int8.linear_i8(x, w, ws, out=torch.empty(4, 31, device=dev)),
           lambda: int8.linear_i8(x, w, ws, out=torch.empty(32, 4, device=dev).t()),
           lambda: int8.gemm_i8(q, s[:3], w, ws), lambda: int8.gemm_i8(q[0], s, w, ws),
           lambda: int8.quantize_i8(x, q=torch.empty(3, 64, dtype=torch.int8, device=dev))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("taken:", i)
    off = torch.empty(33, 64 + 16, dtype=torch.int8, device=dev)
    for f in (lambda: int8.linear_i8(x, off[:, 1:65], torch.ones(33, device=dev)),      # rows not 16-byte aligned
              lambda: int8.quantize_i8(x, q=torch.empty(4, 65, dtype=torch.int8, device=dev)[:, :64]),
              lambda: int8.gemm_i8(torch.empty(1, 131072 + 16, dtype=torch.int8, device=dev), torch.ones(1, device=dev),
                                   torch.empty(1, 131072 + 16, dtype=torch.int8, device=dev), torch.ones(1, device=dev))):
        with pytest.raises(ChimereError) as e:
            f()
        assert e.value.code == 1
    layer = layer_of(4, 32, 64, 1, dev)
    ids, wts = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.ones(4, 2, device=dev)
    for f in (lambda: layer.forward(x, ids.long(), wts), lambda: layer.forward(x, ids[:3], wts[:3]),
              lambda: layer.forward(x, ids, wts[:3]), lambda: layer.forward(x[:, :32], ids, wts),
              lambda: int8.Int8Experts(*(layer.tensors[:4] + [layer.tensors[4].transpose(1, 2), layer.tensors[5]]))):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ChimereError):
        layer.forward(x, torch.zeros(4, 17, dtype=torch.int32, device=dev), torch.ones(4, 17, device=dev))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_address(dev, dtype):
    """Tokens and outputs that start on every element of a vector, rows of odd length, with and without whole vectors."""
    g = gen(3)
    w, ws = weights(301, 515, g)
    for off in range(9):
        print(f"address {off} {dtype}", flush=True)
        for m in (1, 3, 40, 200):
            x = torch.randn(m * 521 + off, generator=g, device=dev).to(TYPES[dtype])[off:].view(m, 521)[:, :515]
            room = torch.full((m * 303 + off,), 7.0, dtype=TYPES[dtype], device=dev)
            int8.linear_i8(x, w, ws, out=room[off:].view(m, 303)[:, :301])
            close(room[off:].view(m, 303)[:, :301], *product(*q_ref(x), w, ws, None, TYPES[dtype]))
            assert (room[:off] == 7.0).all() and (room[off:].view(m, 303)[:, 301:] == 7.0).all()


# ------------------------------------------------------------ offsets past 32 bits

def test_far_outputs(dev):
    """2.4 G outputs: rows on both sides of 2^31 elements."""
    m, n, c = 20000, 120000, 64
    print(f"gemm {m}x{n}x{c}", flush=True)
    g = gen(20)
    a, s = weights(m, c, g)
    w, ws = weights(n, c, g)
    out = int8.gemm_i8(a, s, w, ws, dtype=torch.bfloat16)
    at = torch.tensor([0, 1, 8947, 8948, 17895, 17896, 17897, 19999], device=dev)    # 2^31 / n = 17895.7
    close(out[at], *product(a[at].double().cpu(), s[at].double().cpu(), w, ws, None, torch.bfloat16))


@pytest.mark.parametrize("m", [3, 30, 300])
def test_far_weights(dev, m):
    """Weight rows 64 KB apart, 2.6 GB in all."""
    n, c = 40000, 64
    print(f"gemm far weights {m}", flush=True)
    g = gen(m)
    a, s = weights(m, c, g)
    room = torch.empty(n, 1 << 16, dtype=torch.int8, device=dev)
    room[:, :c], ws = weights(n, c, g)
    w = room[:, :c]
    close(int8.gemm_i8(a, s, w, ws), *product(a.double().cpu(), s.double().cpu(), w, ws, None, torch.float32))


def test_far_rows_of_floats(dev):
    """2.8 G elements in x and bytes in q."""
    n, c = 70000, 40000
    print(f"quantize {n}x{c}", flush=True)
    x = torch.ones(n, c, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, 53687, 53688, 69999], device=dev)
    x[at] = torch.randn(4, c, generator=gen(4), device=dev).to(x.dtype)
    q, s = int8.quantize_i8(x)
    rq, rs = q_ref(x[at])
    assert (q[at].double().cpu() == rq).all() and (s[at].double().cpu() == rs).all()
    assert (q[1] == 127).all() and (q[-2] == 127).all()


@pytest.mark.parametrize("T", [1, 9, 400])
def test_far_experts(dev, T):
    """Experts behind 2^31 bytes of each tensor: as the same experts on their own."""
    E, H, F, n, K = 530, 2048, 2048, 12, 4
    print(f"far experts T={T}", flush=True)
    g = gen(T)
    big, small = [], []
    for rows, cols in ((F, H), (F, H), (H, F)):
        w = torch.empty(E, rows, cols, dtype=torch.int8, device=dev)
        w[-n:] = torch.randint(-128, 128, (n, rows, cols), generator=g, device=dev, dtype=torch.int8)
        s = torch.rand(E, rows, generator=g, device=dev) * 1e-3
        big += [w, s]
        small += [w[-n:].clone(), s[-n:].clone()]
    x = torch.randn(T, H, generator=g, device=dev)
    ids = torch.rand(T, n, generator=g, device=dev).topk(K, 1)[1].to(torch.int32)
    wts = torch.rand(T, K, generator=g, device=dev)
    far = int8.Int8Experts(*big).forward(x, ids + (E - n), wts)
    near = int8.Int8Experts(*small).forward(x, ids, wts)
    assert torch.equal(far, near) and bool(near.abs().sum() > 0)
