"""Root-mean-square norm of the residual stream, the branch's output added to it
before, with an output in floats or in 8 bits for ``int8.gemm_i8``
(``chimere_rms_norm`` / ``chimere_rms_norm_i8`` / ``chimere_rms_norm_grad`` of
include/chimere_hip.h).

    y = rms_norm(x, weight)                             # x [ntok, ncols] float32 / float16 / bfloat16
    y, h = rms_norm(x, weight, residual=stream)         # h = x + stream, y its norm
    q, scale, h = rms_norm_i8(x, weight, residual=stream)
    out = gemm_i8(q, scale, w, w_scale)                 # every product that takes these tokens

The residual has x's type or float32 and h its type; y is formed from the sum
before that rounding.  ``rms_norm`` is recorded for autograd where an input
requires a gradient: its backward pass is ``rms_norm_grad`` at the stored h, in
h's type, and out tensors are refused there, as dual tensors of forward-mode
autograd are always.  A backward pass that is captured
into a graph is captured with its forward pass, and no eager autograd graph of
the same leaves may be alive meanwhile.  Outputs may not overlap inputs, but
``residual_out`` may be the residual.  Stream, device and errors as in
``chimere_amd.int8``.
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import lib
from .int8 import _int8, _out, device_of, empty_i8, float_type, launch, no_tangent, rows_of, vector


def _weight(weight, c):
    """(type, pointer) of a weight of c columns or None."""
    if weight is None:
        return 0, None
    kind = float_type(weight)
    return kind, vector(weight, c, "weight", weight.dtype)


def _residual(x, residual, residual_out, n, c):
    """(type, pointer, stride, out pointer, out stride, h) of the residual, h made where residual_out is None."""
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out without a residual")
        return 0, None, 0, None, 0, None
    kind = float_type(residual)
    if residual.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"residual: {x.dtype} or float32 is wanted, not {residual.dtype}")
    rn, _, ldr = rows_of(residual, "residual", c)
    if rn != n:
        raise ValueError(f"residual: {n} rows are wanted, not {rn}")
    if residual_out is not None and residual_out.dtype != residual.dtype:
        raise ValueError(f"residual_out: {residual.dtype} is wanted, not {residual_out.dtype}")
    h, ldh = _out(residual_out, residual.dtype, n, c, x.device)
    return kind, residual.data_ptr(), ldr, h.data_ptr(), ldh, h


def rms_norm(x, weight=None, eps=1e-6, residual=None, out=None, residual_out=None, dtype=None):
    """y = h * weight / sqrt(mean(h^2) + eps) for each row of h = x (+ residual): y [ntok, ncols] of x's type unless
    ``dtype`` or ``out`` says otherwise, or (y, h) where there is a residual."""
    no_tangent(x, weight, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        if out is not None or residual_out is not None:
            raise ValueError("out and residual_out: not with inputs that require a gradient")
        return _RmsNorm.apply(x, weight, eps, residual, dtype)
    return _rms_norm(x, weight, eps, residual, out, residual_out, dtype)


def _rms_norm(x, weight, eps, residual, out=None, residual_out=None, dtype=None):
    n, c, ld = rows_of(x, "x")
    dev = device_of(x, weight, residual, out, residual_out)
    rtype, res, ldr, hout, ldh, h = _residual(x, residual, residual_out, n, c)
    out, ldo = _out(out, dtype or x.dtype, n, c, x.device)
    launch(dev, lib().chimere_rms_norm, float_type(x), x.data_ptr(), ld, rtype, res, ldr, hout, ldh,
           *_weight(weight, c), eps, float_type(out), out.data_ptr(), ldo, n, c)
    return out if residual is None else (out, h)


def rms_norm_i8(x, weight=None, eps=1e-6, residual=None, q=None, scale=None, residual_out=None):
    """The norm in 8 bits: (q int8 [ntok, ncols], scale float32 [ntok]), and h where there is a residual; y ~ q * scale,
    scale = max |y| / 127 of the row, ties to even.  Not recorded for autograd."""
    n, c, ld = rows_of(x, "x")
    if q is None:
        q = empty_i8(n, c, x.device)
    if scale is None:
        scale = torch.empty(n, dtype=torch.float32, device=x.device)
    qn, _, ldq = _int8(q, "q", c)
    if qn != n:
        raise ValueError(f"q: {n} rows are wanted, not {qn}")
    dev = device_of(x, weight, residual, q, scale, residual_out)
    rtype, res, ldr, hout, ldh, h = _residual(x, residual, residual_out, n, c)
    launch(dev, lib().chimere_rms_norm_i8, float_type(x), x.data_ptr(), ld, rtype, res, ldr, hout, ldh,
           *_weight(weight, c), eps, q.data_ptr(), ldq, vector(scale, n, "scale"), n, c)
    return (q, scale) if residual is None else (q, scale, h)


def rms_norm_grad(h, grad_out, weight=None, eps=1e-6, grad_h=None, out=None, weight_grad=True):
    """(gradient of x and of the residual [ntok, ncols] in h's type, gradient of the weight in the weight's type or
    None) for the gradient ``grad_out`` of y, of any float type; ``grad_h``: what the other uses of h ask, in h's type
    (``out`` may be it)."""
    n, c, ld = rows_of(h, "h")
    gn, _, ldg = rows_of(grad_out, "grad_out", c)
    if gn != n:
        raise ValueError(f"grad_out: {n} rows are wanted, not {gn}")
    ldgh = 0
    if grad_h is not None:
        hn, _, ldgh = rows_of(grad_h, "grad_h", c)
        if hn != n or grad_h.dtype != h.dtype:
            raise ValueError(f"grad_h: {(n, c)} {h.dtype} is wanted, not {(hn, c)} {grad_h.dtype}")
    if out is not None and out.dtype != h.dtype:
        raise ValueError(f"out: {h.dtype} is wanted, not {out.dtype}")
    dev = device_of(h, grad_out, weight, grad_h, out)
    wtype, w = _weight(weight, c)
    out, ldo = _out(out, h.dtype, n, c, h.device)
    gw, need, ws = None, 0, None
    if weight is not None and weight_grad:
        gw = torch.empty_like(weight)
        need = lib().chimere_rms_norm_grad_workspace_size(c, n)
        ws = torch.empty(need, dtype=torch.uint8, device=h.device) if need else None
    launch(dev, lib().chimere_rms_norm_grad, float_type(h), h.data_ptr(), ld, wtype, w, eps, float_type(grad_out),
           grad_out.data_ptr(), ldg, None if grad_h is None else grad_h.data_ptr(), ldgh, out.data_ptr(), ldo,
           None if gw is None else gw.data_ptr(), n, c, None if ws is None else ws.data_ptr(), need)
    return out, gw


def next_to_each_other(t):
    """A gradient whose rows' elements lie next to each other (autograd hands over expanded and transposed ones too)."""
    return t if t is None or t.shape[1] == 1 or t.stride(1) == 1 else t.contiguous()


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual, dtype):
        ctx.set_materialize_grads(False)
        res = _rms_norm(x, weight, eps, residual, dtype=dtype)
        ctx.save_for_backward(x if residual is None else res[1], weight)
        ctx.eps, ctx.x_type, ctx.has_residual = eps, x.dtype, residual is not None
        return res

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_h=None):
        h, weight = ctx.saved_tensors
        need_x, need_w, _, need_r, _ = ctx.needs_input_grad
        gx = gw = None
        if grad_out is not None:
            gx, gw = rms_norm_grad(h, next_to_each_other(grad_out), weight, ctx.eps, next_to_each_other(grad_h),
                                   weight_grad=need_w)
        elif grad_h is not None:
            gx = grad_h
        of_x = gx if gx is None or not need_x else gx.to(ctx.x_type)
        return of_x if need_x else None, gw, None, gx if need_r and ctx.has_residual else None, None


__all__ = ["rms_norm", "rms_norm_grad", "rms_norm_i8"]
