"""What follows a router's choice: its statistics (tokens per expert and the
balance loss, with the gradient of the logits: ``chimere_balance_loss`` /
``chimere_balance_loss_grad`` of include/chimere_hip.h), and its pairs sorted by
expert, the tokens' rows in that order and back, with their gradients
(``chimere_sort_pairs`` / ``chimere_dispatch`` / ``chimere_combine`` /
``chimere_combine_grad``).

The choice itself is ``ggml_gpu.gpu_topk_softmax``.  The counts say which
experts a workload meets (and so which of them to keep on the device where
others stay on the host); the loss is 1 for an even choice and grows up to the
number of experts.

    loss, counts, probs, tokens = balance_loss(logits, ids, mask=mask)
    grad = balance_loss_grad(logits, counts, tokens, grad_loss, ids.shape[1], mask=mask)

Where the logits require a gradient, the loss is recorded for autograd: its
backward pass is ``balance_loss_grad``, with the counts held constant (the
choice has no gradient).  counts, probs and tokens are recorded as constants.
The gradient has the logits' type: in float16 most of a training step's are
below its smallest number (g E / N p (f - d) is near 1e-9), so the loss is
scaled there as any other of such a program.  A backward pass that is captured
into a graph is captured with its forward pass, and no eager autograd graph of
the same leaves may be alive meanwhile.  Stream, device and errors as in
``chimere_amd.int8``.

    pairs = sort_pairs(ids, n_experts, mask=mask)
    rows = dispatch(x, pairs)                           # expert e's: rows[pairs.offsets[e]:pairs.offsets[e + 1]]
    out = combine(product(rows), pairs, wts)            # sum over k of wts[t, k] * the row of pair (t, k)

``dispatch`` takes 8-bit tokens with their scales too, for ``int8.gemm_i8`` on
each expert's rows.  ``dispatch`` and ``combine`` are recorded for autograd
where x, y or the weights require a gradient (x's is ``combine`` of the rows'
gradient without weights, the others' ``combine_grad``), with what is said above
about captured backward passes, and without an out tensor.  Dual tensors of
forward-mode autograd are refused by all three.  Nothing is summed by atomics:
results repeat bit for bit.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import I8, lib
from .int8 import INT_MAX, _int8, _out, device_of, empty_i8, float_type, int_sizes, launch, no_tangent, rows_of, vector
from .norm import next_to_each_other


def _mask(mask, n):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"mask: bool or uint8 is wanted, not {mask.dtype}")
    return vector(mask, n, "mask", mask.dtype)


def balance_loss(logits, ids, mask=None):
    """logits [T, E] float32 / float16 / bfloat16, ids [T, K] int32, mask [T] (0: a token that is left out) ->
    (loss float32 [1], counts int32 [E], probs float32 [E], tokens int32 [1]):
    counts = pairs per expert, probs = mean of softmax(logits), loss = E sum counts / (tokens K) probs.
    The loss alone has a gradient."""
    no_tangent(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _BalanceLoss.apply(logits, ids, mask)
    return _balance_loss(logits, ids, mask)


def _balance_loss(logits, ids, mask):
    n, e, ld = rows_of(logits, "logits")
    ni, k, _ = rows_of(ids, "ids")
    if ni != n:
        raise ValueError(f"ids: {n} rows are wanted, not {ni}")
    device, dev = logits.device, device_of(logits, ids, mask)
    loss = torch.empty(1, dtype=torch.float32, device=device)
    probs = torch.empty(e, dtype=torch.float32, device=device)
    counts = torch.empty(e, dtype=torch.int32, device=device)
    tokens = torch.empty(1, dtype=torch.int32, device=device)
    need = lib().chimere_balance_loss_workspace_size(e, n)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    launch(dev, lib().chimere_balance_loss, float_type(logits), logits.data_ptr(), ld,
           vector(ids, n * k, "ids", torch.int32), k, _mask(mask, n), loss.data_ptr(), probs.data_ptr(),
           counts.data_ptr(), tokens.data_ptr(), e, n, ws.data_ptr() if need else None, need)
    return loss, counts, probs, tokens


def balance_loss_grad(logits, counts, tokens, grad_loss, top_k, mask=None, out=None):
    """Gradient of ``balance_loss`` for the logits, times grad_loss (float32 [1] on the device), in the logits' type."""
    n, e, ld = rows_of(logits, "logits")
    if top_k > INT_MAX:
        int_sizes("top_k", top_k)
    if out is None:
        out = torch.empty(n, e, dtype=logits.dtype, device=logits.device)
    on, oe, ldo = rows_of(out, "out")
    if on != n or oe != e or out.dtype != logits.dtype:
        raise ValueError(f"out: {(n, e)} {logits.dtype} is wanted, not {(on, oe)} {out.dtype}")
    launch(device_of(logits, counts, tokens, grad_loss, mask, out), lib().chimere_balance_loss_grad, float_type(logits),
           logits.data_ptr(), ld, _mask(mask, n), vector(counts, e, "counts", torch.int32),
           vector(tokens, 1, "tokens", torch.int32), vector(grad_loss, 1, "grad_loss"), top_k, out.data_ptr(), ldo, e, n)
    return out


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask):
        loss, counts, probs, tokens = _balance_loss(logits, ids, mask)
        ctx.save_for_backward(logits, counts, tokens, mask)
        ctx.top_k = ids.shape[1]
        ctx.mark_non_differentiable(counts, probs, tokens)
        return loss, counts, probs, tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        logits, counts, tokens, mask = ctx.saved_tensors
        return balance_loss_grad(logits, counts, tokens, grad_loss, ctx.top_k, mask=mask), None, None


class SortedPairs(NamedTuple):
    """A choice's pairs (t, k) by expert: ``order`` int32 [T K], the pair t K + k at each row (-1 behind the last);
    ``position`` int32 [T, K], the row of each pair (-1: it has none); ``offsets`` int32 [E + 1], each expert's first row."""
    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor


MAX_EXPERTS = 1024


def sort_pairs(ids, n_experts, mask=None):
    """ids [T, K] int32, mask [T] (0: a token that is left out) -> SortedPairs, pairs of one expert in their order; an
    id outside [0, n_experts) has no row."""
    n, k, _ = rows_of(ids, "ids")
    if not 0 <= n_experts <= INT_MAX:
        raise ValueError(f"n_experts: {n_experts} is out of range")
    dev, device = device_of(ids, mask), ids.device
    order = torch.empty(n * k, dtype=torch.int32, device=device)
    position = torch.empty(n, k, dtype=torch.int32, device=device)
    # (more experts than MAX_EXPERTS the library refuses: nothing is made for them)
    offsets = torch.empty(min(n_experts, MAX_EXPERTS) + 1, dtype=torch.int32, device=device)
    need = lib().chimere_sort_pairs_workspace_size(n_experts, k, n)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    launch(dev, lib().chimere_sort_pairs, vector(ids, n * k, "ids", torch.int32), _mask(mask, n), order.data_ptr(),
           position.data_ptr(), offsets.data_ptr(), n_experts, k, n, ws.data_ptr() if need else None, need)
    return SortedPairs(order, position, offsets)


def _pairs(pairs):
    """(tokens, top_k, experts, position pointer, offsets pointer) of a SortedPairs."""
    n, k, _ = rows_of(pairs.position, "position")
    e = pairs.offsets.numel() - 1
    return n, k, e, vector(pairs.position, n * k, "position", torch.int32), vector(pairs.offsets, e + 1, "offsets", torch.int32)


SCALES = "scales: with int8 tokens, and with them alone"


def dispatch(x, pairs, scale=None, out=None, out_scale=None):
    """x [T, H] float32 / float16 / bfloat16, or int8 with ``scale`` [T] -> the tokens' rows [T K, H] in the experts'
    order, or (rows, their scales); rows behind the last pair are 0.  An out of fewer rows takes as many."""
    no_tangent(x)
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out: not with an x that requires a gradient")
        if scale is not None or out_scale is not None:
            raise ValueError(SCALES)
        return _Dispatch.apply(x, pairs)
    return _dispatch(x, pairs, scale, out, out_scale)


def _dispatch(x, pairs, scale=None, out=None, out_scale=None):
    eight = x.dtype == torch.int8
    n, c, ld = _int8(x, "x") if eight else rows_of(x, "x")
    t, k, e, position, offsets = _pairs(pairs)
    if t != n:
        raise ValueError(f"x: {t} rows are wanted, not {n}")
    if eight != (scale is not None) or (out_scale is not None and not eight):
        raise ValueError(SCALES)
    if out is not None and out.dtype != x.dtype:
        raise ValueError(f"out: {x.dtype} is wanted, not {out.dtype}")
    if eight:
        out = empty_i8(n * k, c, x.device) if out is None else out
        rows, _, ldo = _int8(out, "out", c)
        out_scale = torch.empty(rows, dtype=torch.float32, device=x.device) if out_scale is None else out_scale
        kind, scales = I8, (vector(scale, n, "scale"), vector(out_scale, rows, "out_scale"))
    else:
        out = torch.empty(n * k, c, dtype=x.dtype, device=x.device) if out is None else out
        rows, _, ldo = rows_of(out, "out", c)
        kind, scales = float_type(x), (None, None)
    launch(device_of(x, pairs.position, pairs.offsets, scale, out, out_scale), lib().chimere_dispatch, kind, x.data_ptr(),
           ld, scales[0], position, offsets, out.data_ptr(), ldo, scales[1], rows, e, k, n, c)
    return (out, out_scale) if eight else out


def _weights(weights, n, k):
    return None if weights is None else vector(weights, n * k, "weights")


def combine(y, pairs, weights=None, out=None, dtype=None):
    """out [T, H] = sum over k, ascending, of weights[t, k] * y[position[t, k]], in f32 and rounded once, of y's type
    unless ``dtype`` or ``out`` says otherwise; weights [T, K] float32, None: 1.  A pair without a row adds nothing."""
    no_tangent(y, weights)
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        if out is not None:
            raise ValueError("out: not with inputs that require a gradient")
        return _Combine.apply(y, weights, pairs, dtype)
    return _combine(y, pairs, weights, out, dtype)


def _combine(y, pairs, weights=None, out=None, dtype=None):
    rows, c, ld = rows_of(y, "y")
    n, k, _, position, _ = _pairs(pairs)
    out, ldo = _out(out, dtype or y.dtype, n, c, y.device)
    launch(device_of(y, pairs.position, pairs.offsets, weights, out), lib().chimere_combine, float_type(y), y.data_ptr(),
           ld, position, _weights(weights, n, k), float_type(out), out.data_ptr(), ldo, rows, k, n, c)
    return out


def combine_grad(grad_out, y, pairs, weights=None, out=None, rows_grad=True, weights_grad=True):
    """(gradient of y in its type, 0 in rows behind the last pair; gradient of the weights [T, K] float32) for the
    gradient ``grad_out`` [T, H] of ``combine``'s output, of any float type; None for one that is not wanted."""
    rows, c, ld = rows_of(y, "y")
    n, k, e, position, offsets = _pairs(pairs)
    gn, _, ldg = rows_of(grad_out, "grad_out", c)
    if gn != n:
        raise ValueError(f"grad_out: {n} rows are wanted, not {gn}")
    if out is not None and (out.dtype != y.dtype or not rows_grad):
        raise ValueError(f"out: {y.dtype} is wanted, not {out.dtype}" if rows_grad else "out without rows_grad")
    ldo = 0
    if rows_grad:
        out, ldo = _out(out, y.dtype, rows, c, y.device)
    gw = torch.empty(n, k, dtype=torch.float32, device=y.device) if weights_grad else None
    launch(device_of(grad_out, y, pairs.position, pairs.offsets, weights, out), lib().chimere_combine_grad,
           float_type(grad_out), grad_out.data_ptr(), ldg, float_type(y), y.data_ptr(), ld, position,
           _weights(weights, n, k), offsets, out.data_ptr() if rows_grad else None, ldo,
           gw.data_ptr() if weights_grad else None, rows, e, k, n, c)
    return out, gw


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pairs):
        ctx.save_for_backward(*pairs)
        return _dispatch(x, pairs)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _combine(next_to_each_other(grad), SortedPairs(*ctx.saved_tensors)), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, pairs, dtype):
        ctx.save_for_backward(y, weights, *pairs)
        return _combine(y, pairs, weights, dtype=dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        y, weights, *pairs = ctx.saved_tensors
        need_y, need_w = ctx.needs_input_grad[:2]
        gy, gw = combine_grad(next_to_each_other(grad), y, SortedPairs(*pairs), weights, rows_grad=need_y, weights_grad=need_w)
        return gy, None if gw is None else gw.view(weights.shape), None, None


__all__ = ["SortedPairs", "balance_loss", "balance_loss_grad", "combine", "combine_grad", "dispatch", "sort_pairs"]
