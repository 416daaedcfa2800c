"""Statistics of a router's choice: tokens per expert and the balance loss,
with the gradient of the logits (``chimere_balance_loss`` /
``chimere_balance_loss_grad`` of include/chimere_hip.h).

The choice itself is ``ggml_gpu.gpu_topk_softmax``.  The counts say which
experts a workload meets (and so which of them to keep on the device where
others stay on the host); the loss is 1 for an even choice and grows up to the
number of experts.

    loss, counts, probs, tokens = balance_loss(logits, ids, mask=mask)
    grad = balance_loss_grad(logits, counts, tokens, grad_loss, ids.shape[1], mask=mask)

Both are plain calls on tensors, to be used from a program's own backward
pass; nothing is recorded for autograd.  Stream, device and errors as in
``chimere_amd.int8``.
"""
import torch

from ._lib import check, lib
from .int8 import _vector, float_type, on_device, rows_of, stream_of


def _mask(mask, n):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"mask: bool or uint8 is wanted, not {mask.dtype}")
    return _vector(mask, n, "mask", mask.dtype)


def balance_loss(logits, ids, mask=None):
    """logits [T, E] float32 / float16 / bfloat16, ids [T, K] int32, mask [T] (0: a token that is left out) ->
    (loss float32 [1], counts int32 [E], probs float32 [E], tokens int32 [1]):
    counts = pairs per expert, probs = mean of softmax(logits), loss = E sum counts / (tokens K) probs."""
    n, e, ld = rows_of(logits, "logits")
    if ids.dim() != 2 or ids.shape[0] != n:
        raise ValueError(f"ids: [{n}, top_k] is wanted, not {tuple(ids.shape)}")
    dev = logits.device
    loss, probs = torch.empty(1, device=dev), torch.empty(e, device=dev)
    counts = torch.empty(e, dtype=torch.int32, device=dev)
    tokens = torch.empty(1, dtype=torch.int32, device=dev)
    with on_device(logits, ids, mask):
        need = lib().chimere_balance_loss_workspace_size(e, n)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        lib().chimere_balance_loss(float_type(logits), logits.data_ptr(), ld,
                                   _vector(ids, ids.numel(), "ids", torch.int32), ids.shape[1], _mask(mask, n),
                                   loss.data_ptr(), probs.data_ptr(), counts.data_ptr(), tokens.data_ptr(), e, n,
                                   ws.data_ptr(), need, stream_of(logits))
    check()
    return loss, counts, probs, tokens


def balance_loss_grad(logits, counts, tokens, grad_loss, top_k, mask=None, out=None):
    """Gradient of ``balance_loss`` for the logits, times grad_loss (float32 [1] on the device), in the logits' type."""
    n, e, ld = rows_of(logits, "logits")
    if out is None:
        out = torch.empty(n, e, dtype=logits.dtype, device=logits.device)
    if out.shape != logits.shape or out.dtype != logits.dtype:
        raise ValueError(f"out: {tuple(logits.shape)} {logits.dtype} is wanted, not {tuple(out.shape)} {out.dtype}")
    _, _, ldo = rows_of(out, "out")
    with on_device(logits, counts, tokens, grad_loss, mask, out):
        lib().chimere_balance_loss_grad(float_type(logits), logits.data_ptr(), ld, _mask(mask, n),
                                        _vector(counts, e, "counts", torch.int32),
                                        _vector(tokens, 1, "tokens", torch.int32), _vector(grad_loss, 1, "grad_loss"),
                                        top_k, out.data_ptr(), ldo, e, n, stream_of(logits))
    check()
    return out


__all__ = ["balance_loss", "balance_loss_grad"]
