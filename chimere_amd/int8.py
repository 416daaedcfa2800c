"""Products over weights in 8-bit integers with one scale per output channel
(``chimere_quantize_i8`` / ``chimere_gemm_i8`` / ``chimere_linear_i8`` /
``chimere_moe_i8`` of include/chimere_hip.h).

    w, w_scale = quantize_i8(weight)              # once; weight [nrows, ncols]
    y = linear_i8(x, w, w_scale)                  # x [ntok, ncols] float32 / float16 / bfloat16

Tokens are quantized within ``linear_i8``; where several matrices take the
same tokens, ``quantize_i8`` once and ``gemm_i8`` for each.  ``Int8Experts``
holds one layer's routed experts in this format.  Outputs may not overlap inputs.

Tensors lie on one ROCm device; launches go to that device's current torch
stream, scratch comes from torch's allocator on it.  Rows of 8-bit integers
start 16-byte aligned: ``quantize_i8`` makes them so (a view of padded rows
where ncols is no multiple of 16).  Nothing is recorded for autograd: these
are the products of a server.  A rejected call raises ``ChimereError``
(the library's checks) or ``ValueError`` (types, shapes, devices).
"""
import ctypes as C

import torch
from torch.autograd import forward_ad

from ._lib import BF16, F16, F32, MoeI8LayerC, check, lib

FLOAT_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def device_of(first, *more):
    """The index of the ROCm device that all tensors (Nones apart) lie on."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError(f"tensors on a ROCm device are wanted, not on {first.device}")
    for t in more:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and on {t.device}")
    return dev


def launch(dev, fn, *args):
    """fn(*args, stream) with device dev's current torch stream, dev being the current device meanwhile."""
    stream = torch._C._cuda_getCurrentRawStream(dev)    # torch.cuda.current_stream(dev).cuda_stream, 1.7 us less
    if dev == torch.cuda.current_device():
        fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            fn(*args, stream)
    check()


def float_type(t):
    kind = FLOAT_TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"float32, float16 or bfloat16 is wanted, not {t.dtype}")
    return kind


def no_tangent(*tensors):
    """Refuses dual tensors of forward-mode autograd where a call has a gradient, but no tangent."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("a tensor with a tangent: forward-mode autograd is not recorded")


INT_MAX = 2 ** 31 - 1


def int_sizes(what, *sizes):
    """Refuses sizes that the C entry points, which take them as int, would see truncated."""
    if max(sizes) > INT_MAX:
        raise ValueError(f"{what}: sizes of at most {INT_MAX} are wanted, not {sizes}")


def rows_of(t, what, ncols=None):
    """(rows, columns, row stride) of a matrix whose rows' elements lie next to each other."""
    if t.dim() != 2:
        raise ValueError(f"{what}: a matrix is wanted, not {tuple(t.shape)}")
    (n, c), (ld, one) = t.shape, t.stride()
    if n > INT_MAX or c > INT_MAX:
        int_sizes(what, n, c)
    if one != 1 and c > 1:
        raise ValueError(f"{what}: contiguous rows are wanted, not {tuple(t.shape)} with strides {t.stride()}")
    if ncols is not None and c != ncols:
        raise ValueError(f"{what}: {c} columns, {ncols} are wanted")
    return n, c, ld if n > 1 else max(ld, c)


def vector(t, n, what, dtype=torch.float32):
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous {dtype} are wanted, not {tuple(t.shape)} {t.dtype}")
    return t.data_ptr()


def _int8(t, what, ncols=None):
    if t.dtype != torch.int8:
        raise ValueError(f"{what}: int8 is wanted, not {t.dtype}")
    n, c, ld = rows_of(t, what, ncols)
    return n, c, ld if n > 1 else (ld + 15) // 16 * 16      # one row has no next one


def _out(out, dtype, n, rows, dev):
    """(out, its row stride), made where it is None."""
    if out is None:
        return torch.empty(n, rows, dtype=dtype, device=dev), rows
    on, oc, ld = rows_of(out, "out")
    if on != n or oc != rows:
        raise ValueError(f"out: {(n, rows)} is wanted, not {(on, oc)}")
    return out, ld


def _bias(bias, n):
    return None if bias is None else vector(bias, n, "bias")


def empty_i8(n, c, device):
    """int8 [n, c], its rows 16-byte aligned."""
    pitch = (c + 15) // 16 * 16
    q = torch.empty(n, pitch, dtype=torch.int8, device=device)
    return q if pitch == c else q[:, :c]


def quantize_i8(x, q=None, scale=None):
    """x [rows, ncols] -> (q int8 [rows, ncols], scale float32 [rows]), x ~ q * scale: scale = max |x| / 127 of the
    row (as torch divides by a number: times 1/127), ties to even.  For tokens and for weights (rows = output channels)."""
    n, c, ld = rows_of(x, "x")
    if q is None:
        q = empty_i8(n, c, x.device)
    if scale is None:
        scale = torch.empty(n, dtype=torch.float32, device=x.device)
    qn, _, ldq = _int8(q, "q", c)
    if qn != n:
        raise ValueError(f"q: {n} rows are wanted, not {qn}")
    launch(device_of(x, q, scale), lib().chimere_quantize_i8, float_type(x), x.data_ptr(), ld, q.data_ptr(), ldq,
           vector(scale, n, "scale"), n, c)
    return q, scale


def gemm_i8(a, a_scale, w, w_scale, bias=None, out=None, dtype=torch.float32):
    """out [ntok, nrows] = (a @ w.T) * a_scale[:, None] * w_scale (+ bias), a [ntok, ncols] and w [nrows, ncols] int8
    with their scales, out of type ``dtype`` unless given."""
    n, c, lda = _int8(a, "a")
    rows, _, ldw = _int8(w, "w", c)
    out, ldo = _out(out, dtype, n, rows, a.device)
    launch(device_of(a, a_scale, w, w_scale, bias, out), lib().chimere_gemm_i8, a.data_ptr(), lda,
           vector(a_scale, n, "a_scale"), w.data_ptr(), ldw, vector(w_scale, rows, "w_scale"), _bias(bias, rows),
           float_type(out), out.data_ptr(), ldo, n, rows, c)
    return out


def linear_i8(x, w, w_scale, bias=None, out=None, dtype=None):
    """``gemm_i8`` of float tokens x [ntok, ncols], quantized within the call; out has x's type unless ``dtype`` or
    ``out`` says otherwise."""
    n, c, ld = rows_of(x, "x")
    rows, _, ldw = _int8(w, "w", c)
    out, ldo = _out(out, dtype or x.dtype, n, rows, x.device)
    dev = device_of(x, w, w_scale, bias, out)
    need = lib().chimere_linear_i8_workspace_size(n, c)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    launch(dev, lib().chimere_linear_i8, float_type(x), x.data_ptr(), ld, w.data_ptr(), ldw,
           vector(w_scale, rows, "w_scale"), _bias(bias, rows), float_type(out), out.data_ptr(), ldo, n, rows, c,
           ws.data_ptr() if need else None, need)
    return out


class Int8Experts:
    """One layer's routed experts: gate, up [E, F, H] and down [E, H, F] int8, their scales [E, F], [E, F] and
    [E, H] float32 (``quantize_i8`` of the matrices' rows).  H and F are multiples of 16."""

    def __init__(self, gate, gate_scale, up, up_scale, down, down_scale):
        if gate.dim() != 3 or up.shape != gate.shape or down.shape != (gate.shape[0], gate.shape[2], gate.shape[1]):
            raise ValueError(f"gate, up [E, F, H] and down [E, H, F] are wanted, not {tuple(gate.shape)}, "
                             f"{tuple(up.shape)}, {tuple(down.shape)}")
        self.E, self.F, self.H = gate.shape
        int_sizes("gate", *gate.shape)
        for name, t in (("gate", gate), ("up", up), ("down", down)):
            if t.dtype != torch.int8 or not t.is_contiguous():
                raise ValueError(f"{name}: contiguous int8 is wanted")
        self.device = device_of(gate, gate_scale, up, up_scale, down, down_scale)
        self.tensors = [gate, gate_scale, up, up_scale, down, down_scale]
        self.c = MoeI8LayerC(self.H, self.F, self.E, gate.data_ptr(), up.data_ptr(), down.data_ptr(),
                             vector(gate_scale, self.E * self.F, "gate_scale"),
                             vector(up_scale, self.E * self.F, "up_scale"),
                             vector(down_scale, self.E * self.H, "down_scale"))
        self.ref = C.byref(self.c)

    @classmethod
    def from_float(cls, gate, up, down):
        """Quantizes float weights gate, up [E, F, H] and down [E, H, F]."""
        parts = []
        for w in (gate, up, down):
            e, r, c = w.shape
            q = torch.empty(e * r, c, dtype=torch.int8, device=w.device)
            _, s = quantize_i8(w.reshape(e * r, c), q)
            parts += [q.view(e, r, c), s.view(e, r)]
        return cls(*parts)

    def forward(self, x, ids, wts, out=None, dtype=None):
        """x [T, H] float, ids [T, K] int32 and wts [T, K] float32 as ``gpu_topk_softmax`` gives them -> out [T, H],
        of x's type unless ``dtype`` or ``out`` says otherwise.  An id outside [0, E) adds nothing."""
        n, _, ld = rows_of(x, "x", self.H)
        out, ldo = _out(out, dtype or x.dtype, n, self.H, x.device)
        ni, k, _ = rows_of(ids, "ids")
        if ni != n:
            raise ValueError(f"ids: {n} rows are wanted, not {ni}")
        if device_of(x, ids, wts, out) != self.device:
            raise ValueError(f"x on {x.device}, the experts on cuda:{self.device}")
        need = lib().chimere_moe_i8_workspace_size(self.ref, k, n)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        launch(self.device, lib().chimere_moe_i8, self.ref, float_type(x), x.data_ptr(), ld,
               vector(ids, n * k, "ids", torch.int32), vector(wts, n * k, "wts"), k, float_type(out), out.data_ptr(),
               ldo, n, ws.data_ptr(), need)
        return out


__all__ = ["Int8Experts", "gemm_i8", "linear_i8", "quantize_i8"]
