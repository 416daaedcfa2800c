"""Routed experts in 8-bit integers with 16-bit outputs: each is the f32 result of the same call, rounded once, whatever
the number of tokens that come with it.  Equalities, so no tolerance but the one of the f32 results' own test."""
import pytest
import torch

from chimere_amd import int8
from test_gpu_int8 import TYPES, close, experts_ref, gen, layer_of, routed

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]

# pairs on their own (8 and 16 columns of the down product, up to 16, 32 and 64 integers of a thread), tiles of 64 and of 128 pairs
SHAPES = [(1, 8, 2, 128, 64), (5, 64, 8, 1024, 1152), (20, 16, 2, 256, 128), (90, 40, 8, 256, 192), (200, 8, 4, 272, 320),
          (700, 16, 16, 192, 512), (3000, 30, 2, 128, 80)]


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("T,E,K,H,F", SHAPES)
def test_rounded_once(dev, T, E, K, H, F):
    g = gen(T + E)
    layer = layer_of(E, F, H, T + K, dev)
    ids, wts = routed(T, E, K, g, dev)
    wts = wts * torch.where(torch.rand(T, K, generator=g, device=dev) < 0.5, -1.0, 1.0)   # experts that cancel
    for name, xt in TYPES.items():
        print(f"experts rounded T={T} E={E} K={K} H={H} F={F} {name}", flush=True)
        x = torch.randn(T, H, generator=g, device=dev).to(xt)
        full = layer.forward(x, ids, wts, dtype=torch.float32)
        for dtype in HALF:
            assert same(layer.forward(x, ids, wts, dtype=dtype), full.to(dtype)), (name, dtype)


@pytest.mark.parametrize("T,E,K,H,F", SHAPES)
def test_against_64_bits(dev, T, E, K, H, F):
    g = gen(T * E)
    layer = layer_of(E, F, H, T + E, dev)
    ids = routed(T, E, K, g, dev)[0]
    wts = torch.randn(T, K, generator=g, device=dev)
    for xt, dtype in ((torch.float16, torch.float16), (torch.float32, torch.float16), (torch.float32, torch.bfloat16),
                      (torch.bfloat16, torch.float32)):
        print(f"experts types T={T} E={E} K={K} H={H} F={F} {xt} {dtype}", flush=True)
        x = torch.randn(T, H, generator=g, device=dev).to(xt)
        close(layer.forward(x, ids, wts, dtype=dtype), *experts_ref(layer, x, ids, wts, dtype))


@pytest.mark.parametrize("dtype", HALF)
def test_as_alone(dev, dtype):
    """A token's row in 16 bits has the same bits alone, in a decode batch and in a chunk."""
    E, K, H, F = 24, 6, 320, 208
    layer, g = layer_of(E, F, H, 3, dev), gen(4)
    x = torch.randn(1500, H, generator=g, device=dev).to(dtype)
    ids, wts = routed(1500, E, K, g, dev)
    full = layer.forward(x, ids, wts)
    for m in (1, 2, 7, 16, 40, 90, 333):
        print(f"experts rows {m} {dtype}", flush=True)
        assert same(layer.forward(x[:m], ids[:m].contiguous(), wts[:m].contiguous()), full[:m]), m


@pytest.mark.parametrize("K,F", [(8, 1152), (8, 2304), (4, 4608), (16, 1024)])
def test_longer_rows_of_h_as_alone(dev, K, F):
    """Rows of h that fill 32 and 64 integers of a thread, five tokens (16 columns at a time) and one (8)."""
    E, H, T = 128, 1024, 5
    g = gen(F)
    w = [torch.randint(-127, 128, (E, r, c), generator=g, device=dev, dtype=torch.int8) for r, c in ((F, H), (F, H), (H, F))]
    s = [torch.rand(E, r, generator=g, device=dev) * 1e-3 + 1e-4 for r in (F, F, H)]
    layer = int8.Int8Experts(w[0], s[0], w[1], s[1], w[2], s[2])
    ids, wts = routed(T, E, K, g, dev)
    x = torch.randn(T, H, generator=g, device=dev)
    print(f"experts longer rows K={K} F={F}", flush=True)
    full = layer.forward(x, ids, wts)
    for t in range(T):
        assert same(layer.forward(x[t:t + 1], ids[t:t + 1], wts[t:t + 1]), full[t:t + 1]), t
    many = layer.forward(x.repeat(60, 1), ids.repeat(60, 1), wts.repeat(60, 1))            # the tiles
    assert same(many[:T], full) and same(many[-T:], full) and bool(full.abs().sum() > 0)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T", [3, 90, 400])
def test_odd_choices(dev, T, dtype):
    """Ids that are no expert, one expert for all, a token without any, a NaN, rows apart: as in f32; what lies around stays."""
    E, K, H, F = 12, 4, 256, 128
    layer, g = layer_of(E, F, H, 9, dev), gen(T)
    x = torch.randn(T, H + 24, generator=g, device=dev).to(dtype)[:, 7:7 + H]
    x[0, 3] = float("nan")
    wts = torch.randn(T, K, generator=g, device=dev)
    for i, ids in enumerate((torch.randint(-3, E + 3, (T, K), generator=g, device=dev), torch.full((T, K), 5, device=dev),
                             torch.full((T, K), -1, device=dev))):
        print(f"experts odd T={T} {dtype} choice {i}", flush=True)
        ids = ids.to(torch.int32)
        ids[1] = -1
        room = torch.full((T, H + 10), 3.0, dtype=dtype, device=dev)
        layer.forward(x, ids, wts, out=room[:, 1:H + 1])
        out = room[:, 1:H + 1]
        assert same(out, layer.forward(x, ids, wts, dtype=torch.float32).to(dtype)) and (out[1] == 0).all()
        assert (room[:, 0] == 3.0).all() and (room[:, H + 1:] == 3.0).all() and not out[1:].isnan().any()


@pytest.mark.parametrize("F", [496, 512, 528, 1024])
def test_largest_sums(dev, F):
    """Rows of h that are all 127 times their scale against columns of -128 and 127, on both sides of F = 516, up to which a
    pair's sums fit 24 bits: a chunk's rows as a token's alone, and the value itself (one rounding each of the sum's
    conversion, two scalings and the weighted sum: 2^-22 of it)."""
    E, K, H = 4, 2, 256
    gate, up = (torch.ones(E, F, H, dtype=torch.int8, device=dev) for _ in range(2))
    down = torch.full((E, H, F), -128, dtype=torch.int8, device=dev)
    down[:, 1::2] = 127
    s = [torch.full((E, r), 2.0 ** -12, device=dev) for r in (F, F, H)]
    layer = int8.Int8Experts(gate, s[0], up, s[1], down, s[2])
    for T in (90, 1500):
        print(f"experts largest sums F={F} T={T}", flush=True)
        x = torch.ones(T, H, device=dev)
        ids = torch.tensor([1, 3], dtype=torch.int32, device=dev).repeat(T, 1)
        wts = torch.tensor([1.0, 0.5], device=dev).repeat(T, 1)
        out, one = layer.forward(x, ids, wts), layer.forward(x[:1], ids[:1], wts[:1])
        assert same(out, one.expand(T, H))
        scale = out[0, 1].double() / (1.5 * 127 * 127 * F)                 # of h's row times that of down
        want = torch.where(torch.arange(H, device=dev) % 2 == 0, -128.0, 127.0).double() * 127 * F * scale * 1.5
        assert bool(((out.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()) and bool((out[:, 0] < 0).all())


@pytest.mark.parametrize("T,F", [(2, 512), (30000, 512), (8000, 1040)])
def test_as_the_calls_one_by_one(dev, T, F):
    """The integers of h are those of silu(g) u in f32 operations that round to nearest each: gate, up and down as products
    of their own and h as torch computes it in between give the same bits.  (An h that is off by a step or two moves a
    few of 15 million integers.)"""
    E, H = 2, 64
    layer, g = layer_of(E, F, H, F, dev), gen(T)
    x = torch.randn(T, H, generator=g, device=dev) * 8
    ids = torch.randint(0, E, (T, 1), generator=g, device=dev).to(torch.int32)
    print(f"experts one by one T={T} F={F}", flush=True)
    out = layer.forward(x, ids, torch.ones(T, 1, device=dev))
    gate, gs, up, us, down, ds = layer.tensors
    for e in range(E):
        q, s = int8.quantize_i8(x)
        a, b = int8.gemm_i8(q, s, gate[e], gs[e]), int8.gemm_i8(q, s, up[e], us[e])
        want = int8.linear_i8(a / (1 + torch.exp(-a)) * b, down[e], ds[e])
        here = ids[:, 0] == e
        assert same(out[here], want[here]), (e, int((out[here] != want[here]).any(1).sum()))
