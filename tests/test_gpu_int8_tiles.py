"""The large tiles of the dense 8-bit integer product over one to many steps of 128 columns, with and without a last part
of a step; and calls on two streams at once, each with its own inputs, bit for bit as alone."""
import pytest
import torch

from chimere_amd import int8
from test_gpu_int8 import TYPES, close, gen, layer_of, product, q_ref, routed, weights

pytestmark = pytest.mark.gpu


# 256 x 256 tiles; 128 x 128 with two stages (512 tiles at most; or more, where a quarter of 256 rows would be empty)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [100, 128, 130, 256, 384, 400, 1100])
@pytest.mark.parametrize("m,n", [(2100, 8200), (1030, 5000), (300, 22000)])
def test_large_tiles(dev, m, n, c, dtype):
    print(f"gemm large {m}x{n}x{c} {dtype}", flush=True)
    g = gen(m + n + c)
    a, s = weights(m, c, g)
    w, ws = weights(n, c, g, pad=16)
    bias = torch.randn(n, generator=g, device=dev) if c % 100 == 0 else None
    out = int8.gemm_i8(a, s, w, ws, bias=bias, dtype=TYPES[dtype])
    rows = torch.cat([torch.arange(0, m, 97), torch.arange(m - 70, m)])       # every tile of rows, the last one whole
    close(out[rows.to(dev)], *product(a[rows.to(dev)].double().cpu(), s[rows.to(dev)].double().cpu(), w, ws, bias, TYPES[dtype]))
    for first in range(0, m, 250):                                            # and all of it, by smaller tiles
        part = int8.gemm_i8(a[first:first + 250], s[first:first + 250], w, ws, bias=bias, dtype=TYPES[dtype])
        assert torch.equal(part, out[first:first + 250]), first


@pytest.mark.parametrize("m,n", [(2100, 8200), (1030, 5000), (300, 22000)])
def test_large_tiles_of_floats(dev, m, n):
    """Float tokens, rows apart on both sides; what lies around the output stays."""
    c = 700
    g = gen(m)
    w, ws = weights(n, c, g)
    for dtype in TYPES.values():
        print(f"linear large {m}x{n}x{c} {dtype}", flush=True)
        x = torch.randn(m, c + 5, generator=g, device=dev).to(dtype)[:, 3:3 + c]
        room = torch.full((m, n + 7), 5.0, dtype=dtype, device=dev)
        int8.linear_i8(x, w, ws, out=room[:, 2:n + 2])
        rows = torch.arange(0, m, 41)
        q, s = q_ref(x[rows.to(dev)])
        close(room[rows.to(dev), 2:n + 2], *product(q, s, w, ws, None, dtype))
        assert (room[:, :2] == 5.0).all() and (room[:, n + 2:] == 5.0).all()


@pytest.mark.parametrize("T", [1, 5, 150, 700])
def test_two_streams_at_once(dev, T):
    """A graph replayed on one stream, eager calls on another, on inputs of their own that no one writes meanwhile."""
    E, K, H, F = 16, 4, 256, 128
    layer, g = layer_of(E, F, H, 2, dev), gen(T)
    w, ws = weights(3000, H, g)

    def inputs():
        return (torch.randn(T, H, generator=g, device=dev),) + routed(T, E, K, g, dev)

    def step(x, ids, wts):
        return layer.forward(x, ids, wts), int8.linear_i8(x, w, ws)

    a, b = inputs(), inputs()
    want_a, want_b = step(*a), step(*b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got_a = step(*a)
    for i in range(10):
        for t in got_a:
            t.fill_(-1.0)
        torch.cuda.synchronize()
        print(f"two streams T={T} round {i}", flush=True)
        with torch.cuda.stream(side):
            others = [step(*b) for _ in range(5)]
        graph.replay()
        more = [step(*a) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for o in others for p, q in zip(o, want_b)), i
        assert all(torch.equal(p, q) for o in more + [got_a] for p, q in zip(o, want_a)), i
