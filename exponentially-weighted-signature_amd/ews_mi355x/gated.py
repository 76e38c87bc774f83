"""Gated linear map of a channel stage (csrc/ews_gated.hip): both projections, the activation and the product in one
kernel (the "glu" and "gelu_glu" stages of ews/block.py:361-374, and their like)."""

from __future__ import annotations

import torch

from . import _native as nat
from .embed import DTYPES, check_tensor, launch, once, refuse_tangents, row_major

_MOST_WIDTH, _MOST_FEATURES = 1 << 16, 1 << 20


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Call:
    """One call's operands as the library takes them; ``gate_weight`` None: the second half of ``weight``'s rows."""

    def __init__(self, x, weight, bias, gate_weight, gate_bias, activation):
        self.x, xs = row_major(x)
        self.weight, ws = row_major(weight)
        self.joint = gate_weight is None
        features = weight.shape[0] // 2 if self.joint else weight.shape[0]
        size = weight.element_size()
        v = self.weight.data_ptr()
        if self.joint:
            g, gs = v + features * ws * size, ws
        else:
            self.gate_weight, gs = row_major(gate_weight)
            g = self.gate_weight.data_ptr()
        self.bias = None if bias is None else bias.contiguous()
        self.gate_bias = None if gate_bias is None else gate_bias.contiguous()
        b, gb = _ptr(self.bias), _ptr(self.gate_bias)
        if self.joint and b is not None:
            gb = b + features * size
        self.desc = nat.GatedDesc(xs, ws, gs, x.shape[0], x.shape[1], features, DTYPES[x.dtype],
                                  nat.GATED_ACTIVATIONS[activation])
        self.at = self.x.data_ptr(), v, g
        self.biases = b, gb

    def workspace(self, call):
        size = nat.load().ews_gated_workspace_bytes(self.desc, *self.at, call)
        return self.x.new_empty(size, dtype=torch.uint8) if size else None

    def forward(self, keep):
        x, v, g = self.at
        b, gb = self.biases
        lib = nat.load()
        out = self.x.new_empty((self.desc.rows, self.desc.features))
        size = lib.ews_gated_kept_bytes(self.desc) if keep else 0
        kept = self.x.new_empty(size, dtype=torch.uint8) if size else None
        ws = self.workspace(nat.GATED_KEEP if keep else nat.GATED_FORWARD)
        nat.check(launch(self.x.device, lib.ews_gated_forward, self.desc, x, v, b, g, gb, out.data_ptr(), _ptr(kept),
                         _ptr(ws)), "ews_gated_forward")
        return out, kept

    def backward(self, kept, gout, needs):
        """The gradients of x, weight, bias, gate_weight and gate_bias that ``needs`` asks for."""
        x, v, g = self.at
        bias, gate_bias = self.biases
        F, H, size = self.desc.features, self.desc.width, self.x.element_size()
        new = self.x.new_empty
        gx = new(self.x.shape) if needs[0] else None
        rows = 2 * F if self.joint else F
        gv, gb = new((rows, H)) if needs[1] else None, new((rows,)) if needs[2] else None
        gg, ggb = new((F, H)) if needs[3] else None, new((F,)) if needs[4] else None
        pv, pb, pg, pgb = _ptr(gv), _ptr(gb), _ptr(gg), _ptr(ggb)
        if self.joint:
            pg = None if gv is None else pv + F * H * size
            pgb = None if gb is None else pb + F * size
        ws = self.workspace(nat.GATED_BACKWARD)
        nat.check(launch(gout.device, nat.load().ews_gated_backward, self.desc, x, v, bias, g, gate_bias, _ptr(kept),
                         gout.data_ptr(), _ptr(gx), pv, pb, pg, pgb, ws.data_ptr()), "ews_gated_backward")
        return gx, gv, gb, gg, ggb


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate_weight, gate_bias, activation):
        call = _Call(x, weight, bias, gate_weight, gate_bias, activation)
        out, kept = call.forward(True)
        ctx.save_for_backward(x, weight, bias, gate_weight, gate_bias, kept)
        ctx.activation = activation
        return out

    @staticmethod
    @once
    def backward(ctx, gout):
        *inputs, kept = ctx.saved_tensors
        call = _Call(*inputs, ctx.activation)
        return (*call.backward(kept, gout.contiguous(), ctx.needs_input_grad), None)


def takes(x, weight, bias):
    """Whether ``gated_linear`` does what a linear map of x and torch's operations after it would, types included."""
    return (x.is_cuda and x.dtype in DTYPES and weight.dtype is x.dtype and weight.device == x.device
            and (bias is None or (bias.dtype is x.dtype and bias.device == x.device))
            and x.shape[-1] == weight.shape[1] and weight.shape[1] <= _MOST_WIDTH
            and weight.shape[0] <= _MOST_FEATURES and not torch.is_autocast_enabled())


def gated_linear(x, weight, bias=None, gate_weight=None, gate_bias=None, activation="sigmoid"):
    """``(x @ V.T + b) * act(x @ G.T + c)``, both products, the activation and the product of the two in one kernel.

    x (..., H) float32 or bfloat16 on the HIP device. weight (2 F, H) and bias (2 F,) hold V's rows and then G's, as a
    joint projection does; with ``gate_weight`` (F, H) given, weight (F, H) and bias (F,) are V and b, gate_weight and
    ``gate_bias`` (F,) G and c. Biases may be None. All of x's type. ``activation``: "sigmoid", "silu", "gelu" (its tanh
    form) or "relu". The result (..., F) is rounded to x's type once.

    Differentiable in everything (reverse mode). A call that records gradients keeps act(g) and v act'(g), of 24 bits
    each (float32: 32), beside the result. Up to 64 rows without gradients (a decoding step) the weights are read once, at the
    memory's rate."""
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
    if H > _MOST_WIDTH or F > _MOST_FEATURES:
        raise ValueError(f"H must be up to {_MOST_WIDTH} and F up to {_MOST_FEATURES}, got {H} and {F}")
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
    if x2.shape[0] == 0:
        none = x.new_zeros(shape)
        return none + sum(t[:0].sum() for t in (x2, *others) if t is not None) if train else none
    if train:
        out = _GatedLinear.apply(x2, *others, activation)
    else:
        out = _Call(x2, *others, activation).forward(False)[0]
    return out if out.shape == shape else out.reshape(shape)
