"""Softmax cross entropy of a linear head without the logits in memory (csrc/ews_loss.hip): the loss end of a
``StackedEWS`` (its seq2seq head with a cross entropy, ews/block.py:695-756)."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as nat
from .embed import DTYPES, check_tensor, launch, row_major


def _desc(hidden, hs, weight, wst, bias, ignore_index, reduction):
    return nat.LossDesc(hs, wst, ignore_index, hidden.shape[0], weight.shape[1], weight.shape[0], DTYPES[weight.dtype],
                        nat.DTYPE_F32 if bias is None else DTYPES[bias.dtype], nat.LOSS_REDUCTIONS[reduction])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run(hidden, weight, bias, targets, ignore_index, reduction, needs, upstream=None, want_loss=True):
    """(loss, [grad_hidden, grad_weight, grad_bias], descriptor); the gradients that ``needs`` asks for, None for the
    others, and no descriptor where there are no rows."""
    lib = nat.load()
    dev = weight.device
    n = hidden.shape[0]
    loss = torch.empty((n,) if reduction == "none" else (), device=dev, dtype=torch.float32) if want_loss else None
    grads = [torch.empty(t.shape, device=dev, dtype=t.dtype) if need else None
             for t, need in zip((hidden, weight, bias), needs)]
    if n == 0:  # no rows: the sum and the mean of nothing are 0
        if loss is not None:
            loss.zero_()
        return loss, [None if g is None else g.zero_() for g in grads], None
    hidden, hs = row_major(hidden)
    weight, wst = row_major(weight)
    bias = None if bias is None else bias.contiguous()
    desc = _desc(hidden, hs, weight, wst, bias, ignore_index, reduction)
    train = any(needs)
    ws = torch.empty(lib.ews_loss_workspace_bytes(desc, int(train)), device=dev, dtype=torch.uint8)
    if train:
        nat.check(launch(dev, lib.ews_loss_train, desc, hidden.data_ptr(), weight.data_ptr(), _ptr(bias),
                         targets.data_ptr(), _ptr(upstream), _ptr(loss), *(_ptr(g) for g in grads), ws.data_ptr()),
                  "ews_loss_train")
    else:
        nat.check(launch(dev, lib.ews_loss_forward, desc, hidden.data_ptr(), weight.data_ptr(), _ptr(bias),
                         targets.data_ptr(), loss.data_ptr(), ws.data_ptr()), "ews_loss_forward")
    return loss, grads, desc


class _LinearCrossEntropy(torch.autograd.Function):
    """The mean and the sum have one upstream number, so their forward computes the gradients with the loss in one pass
    over the rows (ews_loss_train) and the first backward scales them; a second backward of the same graph, and the
    rows' own losses, compute them in the backward."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, ignore_index, reduction):
        ctx.save_for_backward(hidden, weight, bias, targets)
        ctx.args = (ignore_index, reduction)
        needs = ctx.needs_input_grad[:3] if reduction != "none" else (False, False, False)
        loss, grads, ctx.desc = _run(hidden, weight, bias, targets, ignore_index, reduction, needs)
        ctx.grads = grads if any(needs) else None
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        ignore_index, reduction = ctx.args
        if gout.dtype is not torch.float32 or not gout.is_contiguous():
            gout = gout.to(torch.float32).contiguous()
        grads, ctx.grads = ctx.grads, None
        if grads is None:
            hidden, weight, bias, targets = ctx.saved_tensors
            _, grads, ctx.desc = _run(hidden, weight, bias, targets, ignore_index, reduction, ctx.needs_input_grad[:3],
                                      upstream=gout if reduction == "none" else None, want_loss=False)
        if reduction != "none" and ctx.desc is not None:
            nat.check(launch(gout.device, nat.load().ews_loss_scale, ctx.desc, *(_ptr(g) for g in grads),
                             gout.data_ptr()), "ews_loss_scale")
        return (*grads, None, None, None)


def linear_cross_entropy(hidden, weight, targets, bias=None, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits ``hidden @ weight.T + bias`` with whole-number targets, in float32, without the
    logits in memory.

    hidden (..., H) and weight (V, H), both float32 or both bfloat16, bias (V,) of either type or None, targets (...)
    int64 or int32, all on the HIP device. ``reduction``: "mean" over the rows that are not ignored (0 where all are),
    "sum", or "none" for every row's own loss, (...). Differentiable in hidden, weight and bias.

    Rows whose target is ``ignore_index`` have loss and gradient zero, whatever they hold, and cost nothing. A target
    outside [0, V) that is not ``ignore_index`` gives NaN. A bias of -inf takes a token out of the vocabulary."""
    if reduction not in nat.LOSS_REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(nat.LOSS_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (V, H) with V, H >= 1, got {tuple(weight.shape)}")
    V, H = weight.shape
    shape = hidden.shape[:-1]
    if hidden.dim() < 1 or hidden.shape[-1] != H:
        raise ValueError(f"hidden must be (..., {H}), got {tuple(hidden.shape)}")
    if targets.shape != shape:
        raise ValueError(f"targets must be {tuple(shape)}, got {tuple(targets.shape)}")
    if bias is not None and bias.shape != (V,):
        raise ValueError(f"bias must be {(V,)}, got {tuple(bias.shape)}")
    check_tensor("weight", weight)
    check_tensor("hidden", hidden)
    if hidden.dtype is not weight.dtype:
        raise TypeError(f"hidden is {hidden.dtype}, weight {weight.dtype}")
    if bias is not None:
        check_tensor("bias", bias)
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    dev = weight.device
    for name, t in (("hidden", hidden), ("targets", targets), ("bias", bias)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, weight on {dev}")
    rows = hidden if hidden.dim() == 2 else hidden.reshape(-1, H)
    t = targets if targets.dim() == 1 else targets.reshape(-1)
    if t.dtype is not torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        loss = _LinearCrossEntropy.apply(rows, weight, bias, t, int(ignore_index), reduction)
    else:
        loss = _run(rows, weight, bias, t, int(ignore_index), reduction, (False, False, False))[0]
    return loss.reshape(shape) if reduction == "none" and len(shape) != 1 else loss
