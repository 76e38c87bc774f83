"""Losses of a linear head without the logits in memory (csrc/ews_loss.hip): softmax cross entropy, the loss end of a
``StackedEWS`` (its seq2seq head with a cross entropy, ews/block.py:695-756), and distillation from a teacher's largest
logits in its place."""

from __future__ import annotations

import torch

from . import _native as nat
from .embed import DTYPES, check_tensor, launch, once, refuse_tangents, row_major


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Call:
    """One call's operands as the library takes them; ``targets``: the rows' tokens."""

    ABI = "ews_loss_"

    def __init__(self, hidden, weight, bias, reduction, targets, ignore_index):
        self.targets, self.at = targets, (targets.data_ptr(),)
        self.desc = self.head = self._head(hidden, weight, bias, reduction, ignore_index)

    def _head(self, hidden, weight, bias, reduction, ignore_index):
        self.hidden, hs = row_major(hidden)
        self.weight, wst = row_major(weight)
        self.bias = None if bias is None else bias.contiguous()
        self.dev = weight.device
        V, H = weight.shape
        return nat.LossDesc(hs, wst, ignore_index, hidden.shape[0], H, V, DTYPES[weight.dtype],
                            nat.DTYPE_F32 if bias is None else DTYPES[bias.dtype], nat.LOSS_REDUCTIONS[reduction])

    def call(self, name, *args):
        name = self.ABI + name
        nat.check(launch(self.dev, getattr(nat.load(), name), *args), name)

    def keeps(self):
        return getattr(nat.load(), self.ABI + "keeps")(self.desc)

    def workspace(self, train):
        size = getattr(nat.load(), self.ABI + "workspace_bytes_for")(self.desc, self.weight.data_ptr(), train)
        return self.hidden.new_empty(size, dtype=torch.uint8)

    def inputs(self):
        return self.desc, self.hidden.data_ptr(), self.weight.data_ptr(), _ptr(self.bias), *self.at

    def loss(self):
        return self.hidden.new_empty((self.head.rows,) if self.head.reduction == 0 else (), dtype=torch.float32)

    def grads(self, hidden, weight, bias):
        return (self.hidden.new_empty(self.hidden.shape) if hidden else None,
                self.weight.new_empty(self.weight.shape) if weight else None,
                self.bias.new_empty(self.bias.shape) if bias else None)

    def forward(self):
        loss, ws = self.loss(), self.workspace(0)
        self.call("forward", *self.inputs(), loss.data_ptr(), ws.data_ptr())
        return loss

    def train(self, needs, upstream=None, want_loss=True):
        """(loss or None, the gradients that ``needs`` asks for) of one pass over the rows."""
        loss, (gh, gw, gb), ws = self.loss() if want_loss else None, self.grads(*needs), self.workspace(1)
        self.call("train", *self.inputs(), _ptr(upstream), _ptr(loss), _ptr(gh), _ptr(gw), _ptr(gb), ws.data_ptr())
        return loss, (gh, gw, gb)

    def keep(self, need_hidden):
        """The rows' losses, and what ``kept`` forms the gradients from: hidden's and the workspace."""
        loss, gh, ws = self.loss(), self.grads(need_hidden, False, False)[0], self.workspace(1)
        self.call("keep", *self.inputs(), loss.data_ptr(), _ptr(gh), ws.data_ptr())
        return loss, gh, ws

    def kept(self, needs, upstream, gh, ws):
        _, gw, gb = self.grads(False, needs[1], needs[2])
        self.call("kept", self.desc, self.weight.data_ptr(), upstream.data_ptr(), _ptr(gh), _ptr(gw), _ptr(gb),
                  ws.data_ptr())
        return gh, gw, gb


class _DistillCall(_Call):
    """``targets``: a teacher's tokens and logits of every row, and the temperature."""

    ABI = "ews_distill_"

    def __init__(self, hidden, weight, bias, reduction, indices, logits, temperature):
        indices, index_stride = row_major(indices)
        logits, logit_stride = row_major(logits)
        self.targets, self.at = (indices, logits), (indices.data_ptr(), logits.data_ptr())
        self.head = self._head(hidden, weight, bias, reduction, 0)
        self.desc = nat.DistillDesc(self.head, index_stride, logit_stride, indices.shape[1], indices.element_size(),
                                    DTYPES[logits.dtype], temperature)


class _HeadLoss(torch.autograd.Function):
    """The mean and the sum have one upstream number, so their forward computes the gradients with the loss in one pass
    over the rows and the first backward scales them: for an upstream that is no power of two a bfloat16 gradient is
    rounded a second time (float32 until then would be twice the memory, and a pass over it in every step, also in the
    ordinary one whose upstream is 1 and for which nothing is read). The rows' own losses keep the probabilities for the
    first backward, where they fit the scratch (2 GiB). A second backward of the same graph, and the rows' own losses of
    more, compute the probabilities once more.

    ``kind`` is the call's class; ``targets`` and ``args`` are what it takes of targets."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, kind, reduction, args, *targets):
        ctx.save_for_backward(hidden, weight, bias, *targets)
        needs = ctx.needs_input_grad
        call = kind(hidden, weight, bias, reduction, *targets, *args)
        first = None
        if reduction != "none":
            loss, grads = call.train(needs[:3])
            first = call.head, grads
        elif call.keeps():
            loss, *state = call.keep(needs[0])
            first = call, state
        else:
            loss = call.forward()
        ctx.args = first, kind, reduction, args
        return loss

    @staticmethod
    @once
    def backward(ctx, gout):
        first, kind, reduction, args = ctx.args
        ctx.args = None, kind, reduction, args
        none = reduction == "none"
        if gout.dtype is not torch.float32 or not gout.is_contiguous():
            gout = gout.to(torch.float32).contiguous()
        if first is None or none:
            hidden, weight, bias, *targets = ctx.saved_tensors  # refused where one has been changed since
            needs = ctx.needs_input_grad[:3]
            call, state = first or (kind(hidden, weight, bias, reduction, *targets, *args), None)
            head = call.head
            if state:
                grads = call.kept(needs, gout, *state)
            else:
                grads = call.train(needs, upstream=gout if none else None, want_loss=False)[1]
        else:
            head, grads = first
        gh, gw, gb = grads
        if not none:
            nat.check(launch(gout.device, nat.load().ews_loss_scale, head, _ptr(gh), _ptr(gw), _ptr(gb),
                             gout.data_ptr()), "ews_loss_scale")
        return (gh, gw, gb, *[None] * (len(ctx.needs_input_grad) - 3))


def _check_head(hidden, weight, bias, reduction):
    """The checks of a linear head's operands; the rows' shape."""
    if reduction not in nat.LOSS_REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(nat.LOSS_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (V, H) with V, H >= 1, got {tuple(weight.shape)}")
    V, H = weight.shape
    if hidden.dim() < 1 or hidden.shape[-1] != H:
        raise ValueError(f"hidden must be (..., {H}), got {tuple(hidden.shape)}")
    if bias is not None and bias.shape != (V,):
        raise ValueError(f"bias must be {(V,)}, got {tuple(bias.shape)}")
    return hidden.shape[:-1]


def _check_operands(hidden, weight, bias):
    check_tensor("weight", weight)
    check_tensor("hidden", hidden)
    if hidden.dtype is not weight.dtype:
        raise TypeError(f"hidden is {hidden.dtype}, weight {weight.dtype}")
    if bias is not None:
        check_tensor("bias", bias)


def _check_places(dev, names, tensors):
    for name, t in zip(names, tensors):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, weight on {dev}")


def _head_loss(kind, hidden, weight, bias, reduction, args, *targets):
    shape = hidden.shape[:-1]
    rows = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    if rows.shape[0] == 0:  # the sum and the mean of nothing are 0, and so are their gradients
        zero = sum(x[:0].sum(dtype=torch.float32) for x in (rows, weight, bias) if x is not None)
        loss = zero.expand(0) if reduction == "none" else zero
    elif torch.is_grad_enabled() and (rows.requires_grad or weight.requires_grad or
                                      (bias is not None and bias.requires_grad)):
        loss = _HeadLoss.apply(rows, weight, bias, kind, reduction, args, *targets)
    else:
        loss = kind(rows, weight, bias, reduction, *targets, *args).forward()
    return loss.reshape(shape) if reduction == "none" and len(shape) != 1 else loss


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
    return _reduced(rows, kept, reduction)


def _reduced(rows, kept, reduction):
    if reduction == "none":
        return rows
    return rows.sum() / kept.sum().clamp(min=1) if reduction == "mean" else rows.sum()


def logits_distillation(student, indices, logits, temperature, reduction):
    """``linear_distillation`` of a student's logits (..., V) that are in memory, in torch operations, as
    ``logits_cross_entropy`` is of ``linear_cross_entropy``."""
    if reduction not in nat.LOSS_REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(nat.LOSS_REDUCTIONS)}, got {reduction!r}")
    _check_teacher(student.shape[:-1], indices, logits, temperature)
    has = (indices >= 0) & (logits != -float("inf"))
    kept = has.any(-1)
    known = ~(has & (indices >= student.shape[-1])).any(-1)
    at = torch.where(has & (indices < student.shape[-1]), indices, 0).long()
    # in float64: the logarithms cancel at a high temperature, whose square brings out what is left
    teacher = torch.where(has, logits.detach().double() / temperature, -float("inf"))
    logp = torch.log_softmax(torch.where(kept[..., None], teacher, 0.0), -1)
    p = torch.where(has, logp.exp(), 0.0)
    z = torch.where(kept[..., None], student.double(), 0.0)
    logq = torch.log_softmax(z / temperature, -1).gather(-1, at)
    rows = temperature**2 * torch.where(p != 0, p * (logp - logq), 0.0).sum(-1)
    rows = torch.where(kept, rows * torch.where(known, 1.0, float("nan")), 0.0)
    return _reduced(rows, kept, reduction).float()


def _check_teacher(shape, indices, logits, temperature):
    if indices.dim() != len(shape) + 1 or indices.shape[:-1] != shape:
        raise ValueError(f"indices must be {(*shape, 'K')}, got {tuple(indices.shape)}")
    if not 1 <= indices.shape[-1] <= nat.DISTILL_MOST_ENTRIES:
        raise ValueError(f"indices must have 1 to {nat.DISTILL_MOST_ENTRIES} entries a row, got {indices.shape[-1]}")
    if logits.shape != indices.shape:
        raise ValueError(f"logits must be {tuple(indices.shape)}, got {tuple(logits.shape)}")
    if not 1e-6 <= temperature <= 1e4:
        raise ValueError(f"temperature must be from 1e-6 to 1e4, got {temperature}")
    if indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"indices must be int64 or int32, got {indices.dtype}")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise ValueError("the teacher's logits have no gradient here: detach them")


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
    shape = _check_head(hidden, weight, bias, reduction)
    if targets.shape != shape:
        raise ValueError(f"targets must be {tuple(shape)}, got {tuple(targets.shape)}")
    _check_operands(hidden, weight, bias)
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    _check_places(weight.device, ("hidden", "targets", "bias"), (hidden, targets, bias))
    refuse_tangents((hidden, weight, bias))
    t = targets if targets.dim() == 1 else targets.reshape(-1)
    if t.dtype is not torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    return _head_loss(_Call, hidden, weight, bias, reduction, (int(ignore_index),), t)


def linear_distillation(hidden, weight, indices, logits, bias=None, temperature=1.0, reduction="mean"):
    """The distance of a student's distribution from a teacher's largest logits, without the student's logits in
    memory::

        p = softmax(logits / T) over a row's entries     q = softmax((hidden @ weight.T + bias) / T)
        loss = T^2 sum_k p_k (log p_k - log q[indices_k])

    hidden (..., H), weight (V, H) and bias (V,) or None as ``linear_cross_entropy``'s; indices (..., K) int64 or
    int32 and logits (..., K) float32 or bfloat16, K up to 1024: the teacher's tokens of every position and their
    logits, in any order, the teacher's distribution being that over them alone. T is ``temperature`` (1e-6 to 1e4);
    its square keeps the gradients' size. At a high one p and q differ by little: float32's rounding of them, 2^-20 of
    q at most, is T 2^-20 of q in a gradient (1% of a token's at T = 1e4 and logits a unit apart). ``reduction``: "mean"
    over the rows that have an entry (0 where none has), "sum", or "none" for every row's own loss, (...), float32.
    Differentiable in hidden, weight and bias (reverse mode); the teacher's logits have no gradient, and one that
    requires it is refused: detach them.

    An entry with a negative index or a logit of -inf is none: rows may have fewer than K. A row without any has loss
    and gradient zero, whatever it holds, and costs nothing. A token that is named twice is two entries of its
    probabilities. An index of V or more gives NaN. A token that the student's bias has taken out (-inf) and that the
    teacher gives any probability has an infinite loss, and the row's gradients may be NaN. When and how gradients are
    formed is as in ``linear_cross_entropy``."""
    shape = _check_head(hidden, weight, bias, reduction)
    temperature = float(temperature)
    _check_teacher(shape, indices, logits, temperature)
    _check_operands(hidden, weight, bias)
    check_tensor("logits", logits)
    _check_places(weight.device, ("hidden", "indices", "logits", "bias"), (hidden, indices, logits, bias))
    refuse_tangents((hidden, weight, bias, logits))
    K = indices.shape[-1]
    return _head_loss(_DistillCall, hidden, weight, bias, reduction, (temperature,), indices.reshape(-1, K),
                      logits.detach().reshape(-1, K))
