"""Softmax cross entropy of a linear head without the logits in memory (csrc/ews_loss.hip): the loss end of a
``StackedEWS`` (its seq2seq head with a cross entropy, ews/block.py:695-756)."""

from __future__ import annotations

import torch

from . import _native as nat
from .embed import DTYPES, check_tensor, launch, once, refuse_tangents, row_major


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Call:
    """One call's operands as the library takes them."""

    def __init__(self, hidden, weight, bias, targets, ignore_index, reduction):
        self.hidden, hs = row_major(hidden)
        self.weight, wst = row_major(weight)
        self.bias = None if bias is None else bias.contiguous()
        self.targets, self.dev = targets, weight.device
        V, H = weight.shape
        self.desc = nat.LossDesc(hs, wst, ignore_index, hidden.shape[0], H, V, DTYPES[weight.dtype],
                                 nat.DTYPE_F32 if bias is None else DTYPES[bias.dtype], nat.LOSS_REDUCTIONS[reduction])

    def workspace(self, train):
        size = nat.load().ews_loss_workspace_bytes_for(self.desc, self.weight.data_ptr(), train)
        return self.hidden.new_empty(size, dtype=torch.uint8)

    def inputs(self):
        return self.desc, self.hidden.data_ptr(), self.weight.data_ptr(), _ptr(self.bias), self.targets.data_ptr()

    def loss(self):
        return self.hidden.new_empty((self.desc.rows,) if self.desc.reduction == 0 else (), dtype=torch.float32)

    def grads(self, hidden, weight, bias):
        return (self.hidden.new_empty(self.hidden.shape) if hidden else None,
                self.weight.new_empty(self.weight.shape) if weight else None,
                self.bias.new_empty(self.bias.shape) if bias else None)

    def forward(self):
        loss, ws = self.loss(), self.workspace(0)
        nat.check(launch(self.dev, nat.load().ews_loss_forward, *self.inputs(), loss.data_ptr(), ws.data_ptr()),
                  "ews_loss_forward")
        return loss

    def train(self, needs, upstream=None, want_loss=True):
        """(loss or None, the gradients that ``needs`` asks for) of one pass over the rows."""
        loss, (gh, gw, gb), ws = self.loss() if want_loss else None, self.grads(*needs), self.workspace(1)
        nat.check(launch(self.dev, nat.load().ews_loss_train, *self.inputs(), _ptr(upstream), _ptr(loss), _ptr(gh),
                         _ptr(gw), _ptr(gb), ws.data_ptr()), "ews_loss_train")
        return loss, (gh, gw, gb)

    def keep(self, need_hidden):
        """The rows' losses, and what ``kept`` forms the gradients from: hidden's and the workspace."""
        loss, gh, ws = self.loss(), self.grads(need_hidden, False, False)[0], self.workspace(1)
        nat.check(launch(self.dev, nat.load().ews_loss_keep, *self.inputs(), loss.data_ptr(), _ptr(gh), ws.data_ptr()),
                  "ews_loss_keep")
        return loss, gh, ws

    def kept(self, needs, upstream, gh, ws):
        _, gw, gb = self.grads(False, needs[1], needs[2])
        nat.check(launch(self.dev, nat.load().ews_loss_kept, self.desc, self.weight.data_ptr(), upstream.data_ptr(),
                         _ptr(gh), _ptr(gw), _ptr(gb), ws.data_ptr()), "ews_loss_kept")
        return gh, gw, gb


class _LinearCrossEntropy(torch.autograd.Function):
    """The mean and the sum have one upstream number, so their forward computes the gradients with the loss in one pass
    over the rows and the first backward scales them: for an upstream that is no power of two a bfloat16 gradient is
    rounded a second time (float32 until then would be twice the memory, and a pass over it in every step, also in the
    ordinary one whose upstream is 1 and for which nothing is read). The rows' own losses keep the probabilities for the
    first backward, where they fit the scratch (2 GiB). A second backward of the same graph, and the rows' own losses of
    more, compute the probabilities once more."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, ignore_index, reduction):
        ctx.save_for_backward(hidden, weight, bias, targets)
        needs = ctx.needs_input_grad
        call = _Call(hidden, weight, bias, targets, ignore_index, reduction)
        first = None
        if reduction != "none":
            loss, grads = call.train(needs[:3])
            first = call.desc, grads
        elif nat.load().ews_loss_keeps(call.desc):
            loss, *state = call.keep(needs[0])
            first = call, state
        else:
            loss = call.forward()
        ctx.args = first, ignore_index, reduction
        return loss

    @staticmethod
    @once
    def backward(ctx, gout):
        first, ignore_index, reduction = ctx.args
        ctx.args = None, ignore_index, reduction
        none = reduction == "none"
        if gout.dtype is not torch.float32 or not gout.is_contiguous():
            gout = gout.to(torch.float32).contiguous()
        if first is None or none:
            inputs = ctx.saved_tensors  # refused where one has been changed since
            needs = ctx.needs_input_grad[:3]
            call, state = first or (_Call(*inputs, ignore_index, reduction), None)
            desc = call.desc
            if state:
                grads = call.kept(needs, gout, *state)
            else:
                grads = call.train(needs, upstream=gout if none else None, want_loss=False)[1]
        else:
            desc, grads = first
        gh, gw, gb = grads
        if not none:
            nat.check(launch(gout.device, nat.load().ews_loss_scale, desc, _ptr(gh), _ptr(gw), _ptr(gb),
                             gout.data_ptr()), "ews_loss_scale")
        return gh, gw, gb, None, None, None


def logits_cross_entropy(logits, targets, ignore_index, reduction):
    """``linear_cross_entropy`` of logits (..., V) that are in memory, in torch operations: for a head that is more than
    a linear map. Ignored rows and targets outside the vocabulary are answered alike."""
    if reduction not in nat.LOSS_REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(nat.LOSS_REDUCTIONS)}, got {reduction!r}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets must be {tuple(logits.shape[:-1])}, got {tuple(targets.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    kept = targets != ignore_index
    known = (targets >= 0) & (targets < logits.shape[-1])
    z = torch.where(kept[..., None], logits.float(), 0.0)
    at = torch.where(known, targets, 0).long()
    rows = -torch.log_softmax(z, -1).gather(-1, at[..., None])[..., 0]
    rows = torch.where(kept, rows * torch.where(known | ~kept, 1.0, float("nan")), 0.0)
    if reduction == "none":
        return rows
    return rows.sum() / kept.sum().clamp(min=1) if reduction == "mean" else rows.sum()


def linear_cross_entropy(hidden, weight, targets, bias=None, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits ``hidden @ weight.T + bias`` with whole-number targets, in float32, without the
    logits in memory.

    hidden (..., H) and weight (V, H), both float32 or both bfloat16, bias (V,) of either type or None, targets (...)
    int64 or int32, all on the HIP device. ``reduction``: "mean" over the rows that are not ignored (0 where all are),
    "sum", or "none" for every row's own loss, (...). Differentiable in hidden, weight and bias (reverse mode).

    Where a gradient is required the mean and the sum form it with the loss, three products for one: a validation loss
    is best taken under ``torch.no_grad``. bfloat16 gradients are rounded once where the upstream number of the mean or
    the sum is a power of two (1 as a rule), else a second time after the multiplication by it.

    Rows whose target is ``ignore_index`` have loss and gradient zero, whatever they hold, and cost nothing. A target
    outside [0, V) that is not ``ignore_index`` gives NaN. A bias of -inf takes a token out of the vocabulary, and so
    does a logit of -inf from an infinite weight; a row with a logit of +inf or NaN has a loss of NaN. A row whose
    target has been taken out has an infinite loss, and its gradients may be NaN."""
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
    refuse_tangents((hidden, weight, bias))
    rows = hidden if hidden.dim() == 2 else hidden.reshape(-1, H)
    t = targets if targets.dim() == 1 else targets.reshape(-1)
    if t.dtype is not torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    if rows.shape[0] == 0:  # the sum and the mean of nothing are 0, and so are their gradients
        zero = sum(x[:0].sum(dtype=torch.float32) for x in (rows, weight, bias) if x is not None)
        loss = zero.expand(0) if reduction == "none" else zero
    elif torch.is_grad_enabled() and (rows.requires_grad or weight.requires_grad or
                                      (bias is not None and bias.requires_grad)):
        loss = _LinearCrossEntropy.apply(rows, weight, bias, t, int(ignore_index), reduction)
    else:
        loss = _Call(rows, weight, bias, t, int(ignore_index), reduction).forward()
    return loss.reshape(shape) if reduction == "none" and len(shape) != 1 else loss
