"""Products over weights in 8-bit integers with one scale per output channel
(``chimere_quantize_i8`` / ``chimere_gemm_i8`` / ``chimere_linear_i8`` /
``chimere_moe_i8`` of include/chimere_hip.h).

    w, w_scale = quantize_i8(weight)              # once; weight [nrows, ncols]
    y = linear_i8(x, w, w_scale)                  # x [ntok, ncols] float32 / float16 / bfloat16

Tokens are quantized within ``linear_i8``; where several matrices take the
same tokens, ``quantize_i8`` once and ``gemm_i8`` for each.  ``Int8Experts``
holds one layer's routed experts in this format.

Tensors lie on one ROCm device; launches go to that device's current torch
stream, scratch comes from torch's allocator on it.  Rows of 8-bit integers
start 16-byte aligned: ``quantize_i8`` makes them so (a view of padded rows
where ncols is no multiple of 16).  A rejected call raises ``ChimereError``
(the library's checks) or ``ValueError`` (types, shapes, devices).
"""
import ctypes as C

import torch

from ._lib import BF16, F16, F32, MoeI8LayerC, check, lib

FLOAT_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def on_device(*tensors):
    """The device that all tensors (Nones apart) lie on, as a guard for the launch."""
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"tensors on a ROCm device are wanted, not on {dev}")
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on {dev} and on {t.device}")
    return torch.cuda.device(dev)


def float_type(t):
    if t.dtype not in FLOAT_TYPES:
        raise ValueError(f"float32, float16 or bfloat16 is wanted, not {t.dtype}")
    return FLOAT_TYPES[t.dtype]


def rows_of(t, what, ncols=None):
    """(rows, columns, row stride) of a matrix whose rows' elements lie next to each other."""
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{what}: a matrix with contiguous rows is wanted, not {tuple(t.shape)} strides {t.stride()}")
    if ncols is not None and t.shape[1] != ncols:
        raise ValueError(f"{what}: {t.shape[1]} columns, {ncols} are wanted")
    return t.shape[0], t.shape[1], t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _vector(t, n, what, dtype=torch.float32):
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous {dtype} are wanted, not {tuple(t.shape)} {t.dtype}")
    return t.data_ptr()


def _int8(t, what, ncols=None):
    if t.dtype != torch.int8:
        raise ValueError(f"{what}: int8 is wanted, not {t.dtype}")
    n, c, ld = rows_of(t, what, ncols)
    return n, c, ld if n > 1 else (max(ld, c) + 15) // 16 * 16


def _out(out, dtype, n, rows, dev):
    if out is None:
        return torch.empty(n, rows, dtype=dtype, device=dev)
    if out.shape != (n, rows):
        raise ValueError(f"out: {(n, rows)} is wanted, not {tuple(out.shape)}")
    return out


def stream_of(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def quantize_i8(x, q=None, scale=None):
    """x [rows, ncols] -> (q int8 [rows, ncols], scale float32 [rows]), x ~ q * scale: scale = max |x| / 127 of the
    row, ties to even.  For tokens and for weights (rows = output channels)."""
    n, c, ld = rows_of(x, "x")
    if q is None:
        q = torch.empty(n, (c + 15) // 16 * 16, dtype=torch.int8, device=x.device)[:, :c]
    if scale is None:
        scale = torch.empty(n, dtype=torch.float32, device=x.device)
    qn, _, ldq = _int8(q, "q", c)
    if qn != n:
        raise ValueError(f"q: {n} rows are wanted, not {qn}")
    with on_device(x, q, scale):
        lib().chimere_quantize_i8(float_type(x), x.data_ptr(), ld, q.data_ptr(), ldq, _vector(scale, n, "scale"), n, c,
                                  stream_of(x))
    check()
    return q, scale


def gemm_i8(a, a_scale, w, w_scale, bias=None, out=None, dtype=torch.float32):
    """out [ntok, nrows] = (a @ w.T) * a_scale[:, None] * w_scale (+ bias), a [ntok, ncols] and w [nrows, ncols] int8
    with their scales, out of type ``dtype`` unless given."""
    n, c, lda = _int8(a, "a")
    rows, _, ldw = _int8(w, "w", c)
    out = _out(out, dtype, n, rows, a.device)
    _, _, ldo = rows_of(out, "out")
    with on_device(a, a_scale, w, w_scale, bias, out):
        lib().chimere_gemm_i8(a.data_ptr(), lda, _vector(a_scale, n, "a_scale"), w.data_ptr(), ldw,
                              _vector(w_scale, rows, "w_scale"),
                              None if bias is None else _vector(bias, rows, "bias"), float_type(out), out.data_ptr(),
                              ldo, n, rows, c, stream_of(a))
    check()
    return out


def linear_i8(x, w, w_scale, bias=None, out=None, dtype=None):
    """``gemm_i8`` of float tokens x [ntok, ncols], quantized within the call; out has x's type unless ``dtype`` or
    ``out`` says otherwise."""
    n, c, ld = rows_of(x, "x")
    rows, _, ldw = _int8(w, "w", c)
    out = _out(out, dtype or x.dtype, n, rows, x.device)
    _, _, ldo = rows_of(out, "out")
    with on_device(x, w, w_scale, bias, out):
        need = lib().chimere_linear_i8_workspace_size(n, c)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        lib().chimere_linear_i8(float_type(x), x.data_ptr(), ld, w.data_ptr(), ldw, _vector(w_scale, rows, "w_scale"),
                                None if bias is None else _vector(bias, rows, "bias"), float_type(out), out.data_ptr(),
                                ldo, n, rows, c, ws.data_ptr(), need, stream_of(x))
    check()
    return out


class Int8Experts:
    """One layer's routed experts: gate, up [E, F, H] and down [E, H, F] int8, their scales [E, F], [E, F] and
    [E, H] float32 (``quantize_i8`` of the matrices' rows).  H and F are multiples of 16."""

    def __init__(self, gate, gate_scale, up, up_scale, down, down_scale):
        if gate.dim() != 3 or up.shape != gate.shape or down.shape != (gate.shape[0], gate.shape[2], gate.shape[1]):
            raise ValueError(f"gate, up [E, F, H] and down [E, H, F] are wanted, not {tuple(gate.shape)}, "
                             f"{tuple(up.shape)}, {tuple(down.shape)}")
        self.E, self.F, self.H = gate.shape
        for name, t in (("gate", gate), ("up", up), ("down", down)):
            if t.dtype != torch.int8 or not t.is_contiguous():
                raise ValueError(f"{name}: contiguous int8 is wanted")
        on_device(gate, gate_scale, up, up_scale, down, down_scale)
        self.device = gate.device
        self.tensors = [gate, gate_scale, up, up_scale, down, down_scale]
        self.c = MoeI8LayerC(self.H, self.F, self.E, gate.data_ptr(), up.data_ptr(), down.data_ptr(),
                             _vector(gate_scale, self.E * self.F, "gate_scale"),
                             _vector(up_scale, self.E * self.F, "up_scale"),
                             _vector(down_scale, self.E * self.H, "down_scale"))

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
        out = _out(out, dtype or x.dtype, n, self.H, x.device)
        _, _, ldo = rows_of(out, "out")
        if ids.dim() != 2 or ids.shape[0] != n:
            raise ValueError(f"ids: [{n}, top_k] is wanted, not {tuple(ids.shape)}")
        k = ids.shape[1]
        with on_device(self.tensors[0], x, ids, wts, out):
            need = lib().chimere_moe_i8_workspace_size(C.byref(self.c), k, n)
            ws = torch.empty(need, dtype=torch.uint8, device=x.device)
            lib().chimere_moe_i8(C.byref(self.c), float_type(x), x.data_ptr(), ld,
                                 _vector(ids, n * k, "ids", torch.int32), _vector(wts, n * k, "wts"), k,
                                 float_type(out), out.data_ptr(), ldo, n, ws.data_ptr(), need, stream_of(x))
        check()
        return out


__all__ = ["Int8Experts", "gemm_i8", "linear_i8", "quantize_i8"]
