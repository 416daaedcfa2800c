"""Statistics of a router's choice: tokens per expert and the balance loss,
with the gradient of the logits (``chimere_balance_loss`` /
``chimere_balance_loss_grad`` of include/chimere_hip.h).

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
"""
import torch
from torch.autograd.function import once_differentiable

from ._lib import lib
from .int8 import INT_MAX, device_of, float_type, int_sizes, launch, rows_of, vector


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


__all__ = ["balance_loss", "balance_loss_grad"]
