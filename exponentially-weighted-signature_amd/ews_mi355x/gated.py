"""Gated linear map of a channel stage (csrc/ews_gated.hip): both projections, the activation and the product in one
kernel (the "glu" and "gelu_glu" stages of ews/block.py:361-374, and their like)."""

from __future__ import annotations

import torch
from torch._C._functorch import is_batchedtensor, is_legacy_batchedtensor
from torch.nn.functional import linear

from . import _native as nat
from .embed import (DTYPES, aligned, check_tensor, has_tangent, launch, once, refuse_tangents, returned,
                    row_major)

_MOST_ROWS, _MOST_WIDTH, _MOST_FEATURES = 1 << 24, 1 << 16, 1 << 20


def _fits(N, H, F):
    """Whether the library takes these sizes."""
    Np, Hp, ld = (-(-n // 64) * 64 for n in (N, H, F))
    return (N <= _MOST_ROWS and H <= _MOST_WIDTH and F <= _MOST_FEATURES
            and max(Np, F) * Hp <= 1 << 33 and Np * ld <= 1 << 34)


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Call:
    """One call's operands as the library takes them (copies only where rows are not contiguous); ``gate_weight`` None:
    the second half of ``weight``'s rows. A backward whose operands lie where its forward's did is given the forward's
    descriptor: a small call costs its host time, and the backward's thread runs Python two to three times slower than
    the caller's."""

    __slots__ = ("operands", "desc", "at")

    def __init__(self, operands, desc=None, activation=None):
        x, weight, bias, gate_weight, gate_bias = operands
        joint = gate_weight is None
        if desc is None:
            x, xs = row_major(x)
            weight, ws = row_major(weight)
            gs = ws
            if not joint:
                gate_weight, gs = row_major(gate_weight)
            if bias is not None:
                bias = bias.contiguous()
            if gate_bias is not None:
                gate_bias = gate_bias.contiguous()
            desc = nat.GatedDesc(xs, ws, gs, x.shape[0], x.shape[1], weight.shape[0] // 2 if joint else weight.shape[0],
                                 DTYPES[x.dtype], nat.GATED_ACTIVATIONS[activation])
            operands = x, weight, bias, gate_weight, gate_bias
        self.operands, self.desc = operands, desc
        v, b = weight.data_ptr(), _ptr(bias)
        if joint:
            size = 4 if desc.dtype == nat.DTYPE_F32 else 2
            g = v + desc.features * desc.weight_stride * size
            gb = None if b is None else b + desc.features * size
        else:
            g, gb = gate_weight.data_ptr(), _ptr(gate_bias)
        self.at = x.data_ptr(), v, b, g, gb  # what the library is given of them

    def scratch_bytes(self, call):
        x, v, _, g, _ = self.at
        return nat.load().ews_gated_workspace_bytes(self.desc, x, v, g, call)

    def forward(self, keep):
        x = self.operands[0]
        lib = nat.load()
        out = x.new_empty((self.desc.rows, self.desc.features))
        kept = _scratch(x, lib.ews_gated_kept_bytes(self.desc)) if keep else None
        ws = _scratch(x, self.scratch_bytes(nat.GATED_KEEP if keep else nat.GATED_FORWARD))
        nat.check(launch(x.device, lib.ews_gated_forward, self.desc, *self.at, out.data_ptr(), _ptr(kept), _ptr(ws)),
                  "ews_gated_forward")
        return out, kept

    def backward(self, kept, gout, needs, scratch_bytes):
        """The gradients of x, weight, bias, gate_weight and gate_bias that ``needs`` asks for."""
        x, weight, _, gate_weight, _ = self.operands
        F, H = self.desc.features, self.desc.width
        new = x.new_empty
        gx = new(x.shape) if needs[0] else None
        gv = new(weight.shape) if needs[1] else None
        gb = new((weight.shape[0],)) if needs[2] else None
        gg = new(weight.shape) if needs[3] else None
        ggb = new((F,)) if needs[4] else None
        pv, pb = _ptr(gv), _ptr(gb)
        if gate_weight is None:
            size = 4 if self.desc.dtype == nat.DTYPE_F32 else 2
            pg = None if pv is None else pv + F * H * size
            pgb = None if pb is None else pb + F * size
        else:
            pg, pgb = _ptr(gg), _ptr(ggb)
        ws = _scratch(x, scratch_bytes)
        nat.check(launch(gout.device, nat.load().ews_gated_backward, self.desc, *self.at, _ptr(kept), gout.data_ptr(),
                         _ptr(gx), pv, pb, pg, pgb, ws.data_ptr()), "ews_gated_backward")
        return gx, gv, gb, gg, ggb


def _scratch(x, size):
    return x.new_empty(size, dtype=torch.uint8) if size else None


def _come_back(operands, kept, desc, dtype, dev):
    """Saved tensors that are not where the forward left them."""
    N, H, F = desc.rows, desc.width, desc.features
    rows = 2 * F if operands[3] is None else F
    shapes = (N, H), (rows, H), (rows,), (F, H), (F,)
    size = nat.load().ews_gated_kept_bytes(desc)
    operands = [returned(t, dtype, s, dev) for t, s in zip(operands, shapes)]
    return operands, aligned(returned(kept, torch.uint8, (size,), dev))


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate_weight, gate_bias, activation):
        call = _Call((x, weight, bias, gate_weight, gate_bias), activation=activation)
        out, kept = call.forward(True)
        ctx.save_for_backward(*call.operands, kept)
        x, weight, _, gate_weight, _ = call.operands
        ctx.args = (call.desc, call.scratch_bytes(nat.GATED_BACKWARD), activation, call.at, _ptr(kept), x.stride(),
                    weight.stride(), gate_weight is not None and gate_weight.stride(), x.dtype)
        return out

    @staticmethod
    @once
    def backward(ctx, gout):
        *operands, kept = ctx.saved_tensors
        desc, size, activation, at, left, x_strides, strides, gate_strides, dtype = ctx.args
        x, weight, _, gate_weight, _ = operands
        call = _Call(operands, desc)
        if (call.at != at or (left and kept.data_ptr() != left) or x.stride() != x_strides or weight.stride() != strides
                or (gate_strides and gate_weight.stride() != gate_strides) or x.dtype is not dtype
                or weight.dtype is not dtype):
            operands, kept = _come_back(operands, kept, desc, dtype, gout.device)
            call = _Call(operands, activation=activation)
            size = call.scratch_bytes(nat.GATED_BACKWARD)
        return (*call.backward(kept, gout.contiguous(), ctx.needs_input_grad, size), None)


class _GatedStage(_GatedLinear):
    """``_GatedLinear`` with the activation "sigmoid" and, in torch's operations, a graph of its backward and a backward
    of many upstream gradients at a time (``is_grads_batched``)."""

    @staticmethod
    def forward(ctx, x, weight, bias, gate_weight, gate_bias, activation):
        out = _GatedLinear.forward(ctx, x, weight, bias, gate_weight, gate_bias, activation)
        # what came in: a copy that the library took has no graph (the backward then makes it once more)
        ctx.save_for_backward(x, weight, bias, gate_weight, gate_bias, ctx.to_save[-1])
        return out

    @staticmethod
    def backward(ctx, gout):
        graph = torch.is_grad_enabled()
        if not (graph or is_legacy_batchedtensor(gout) or is_batchedtensor(gout)):
            return _GatedLinear.backward(ctx, gout)
        needs = ctx.needs_input_grad[:5]
        with torch.enable_grad():
            x, weight, bias, gate_weight, gate_bias = leaves = [t if t is None else t.view_as(t)
                                                                for t in ctx.saved_tensors[:5]]
            if gate_weight is None:
                v, g = linear(x, weight, bias).chunk(2, -1)
            else:
                v, g = linear(x, weight, bias), linear(x, gate_weight, gate_bias)
            y = v * torch.sigmoid(g)
        grads = iter(torch.autograd.grad(y, [t for t, n in zip(leaves, needs) if n], gout, create_graph=graph))
        return (*(next(grads) if n else None for n in needs), None)


def takes(x, weight, bias):
    """Whether ``gated_linear`` does what a linear map of x and torch's operations after it would, types included."""
    return (x.is_cuda and x.dtype in DTYPES and weight.dtype is x.dtype and weight.device == x.device
            and (bias is None or (bias.dtype is x.dtype and bias.device == x.device))
            and x.shape[-1] == weight.shape[1] and _fits(x.numel() // x.shape[-1], weight.shape[1], weight.shape[0])
            and not torch.is_autocast_enabled() and not has_tangent((x, weight, bias)))


def gated_stage(x, weight, bias=None, gate_weight=None, gate_bias=None):
    """``gated_linear`` for a block's gated channel stage, whose maps have second derivatives: a graph of the backward
    is that of the maps' own."""
    return _gated(_GatedStage, x, weight, bias, gate_weight, gate_bias, "sigmoid")


def gated_linear(x, weight, bias=None, gate_weight=None, gate_bias=None, activation="sigmoid"):
    """``(x @ V.T + b) * act(x @ G.T + c)``, both products, the activation and the product of the two in one kernel.

    x (..., H) float32 or bfloat16 on the HIP device. weight (2 F, H) and bias (2 F,) hold V's rows and then G's, as a
    joint projection does; with ``gate_weight`` (F, H) given, weight (F, H) and bias (F,) are V and b, gate_weight and
    ``gate_bias`` (F,) G and c. Biases may be None. All of x's type. ``activation``: "sigmoid", "silu", "gelu" (its tanh
    form) or "relu". The result (..., F) is rounded to x's type once.

    Differentiable in everything (reverse mode). A call that records gradients keeps both products' sums, of 24
    bits each (float32: 32), beside the result, unless H and F are 64 at most. A few rows (a decoding step:
    32, of float32 64) read the weights once, at the memory's rate."""
    return _gated(_GatedLinear, x, weight, bias, gate_weight, gate_bias, activation)


def _gated(function, x, weight, bias, gate_weight, gate_bias, activation):
    if activation not in nat.GATED_ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(nat.GATED_ACTIVATIONS)}, got {activation!r}")
    joint = gate_weight is None
    if weight.dim() != 2 or weight.numel() == 0 or (joint and weight.shape[0] % 2):
        raise ValueError(f"weight must be {'(2 F, H)' if joint else '(F, H)'} with F, H >= 1, got "
                         f"{tuple(weight.shape)}")
    rows, H = weight.shape
    F = rows // 2 if joint else rows
    if x.dim() < 1 or x.shape[-1] != H:
        raise ValueError(f"x must be (..., {H}), got {tuple(x.shape)}")
    if not joint and gate_weight.shape != weight.shape:
        raise ValueError(f"gate_weight must be {tuple(weight.shape)}, got {tuple(gate_weight.shape)}")
    if joint and gate_bias is not None:
        raise ValueError("gate_bias goes with gate_weight: a joint weight's bias holds both")
    if bias is not None and bias.shape != (rows,):
        raise ValueError(f"bias must be {(rows,)}, got {tuple(bias.shape)}")
    if gate_bias is not None and gate_bias.shape != (F,):
        raise ValueError(f"gate_bias must be {(F,)}, got {tuple(gate_bias.shape)}")
    N = x.numel() // H
    if not _fits(N, H, F):
        raise ValueError(f"up to {_MOST_ROWS} rows, H up to {_MOST_WIDTH} and F up to {_MOST_FEATURES}, and, padded to "
                         f"whole 64s, rows * H and F * H up to 2^33 and rows * F up to 2^34, got {N}, {H} and {F}")
    check_tensor("x", x)
    others = weight, bias, gate_weight, gate_bias
    for name, t in zip(("weight", "bias", "gate_weight", "gate_bias"), others):
        if t is None:
            continue
        if t.dtype is not x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x {x.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    refuse_tangents((x, *others))
    shape = (*x.shape[:-1], F)
    x2 = x if x.dim() == 2 else x.reshape(-1, H)
    train = torch.is_grad_enabled() and (x.requires_grad or any(t is not None and t.requires_grad for t in others))
    if N == 0:
        none = x.new_zeros(shape)
        return none + sum(t[:0].sum() for t in (x2, *others) if t is not None) if train else none
    if train:
        out = function.apply(x2, *others, activation)
    else:
        out = _Call((x2, *others), activation=activation).forward(False)[0]
    return out if out.shape == shape else out.reshape(shape)
