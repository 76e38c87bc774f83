"""Gated linear recurrence over sequences (csrc/ews_gated_scan.hip): per channel and step a decay of its own, where the
depth-1 scans of ``EWS`` have a generator and a clock (the reference writes such recurrences as depth-1 EWS,
ews/conversion/reference/recurrences.py:48-113)."""

from __future__ import annotations

import torch
from torch.autograd.graph import increment_version

from . import _native as nat
from .embed import DTYPES, aligned, check_tensor, launch, once, refuse_tangents, returned
from .gated import _scratch


def _ptr(t):
    return None if t is None else t.data_ptr()


def _neighbours(t):
    """t with its channels next to each other (a copy only where they are not)."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _touches(t, start, end):
    """Whether t lies in the bytes from start to end, in part."""
    first = t.data_ptr()
    if first >= end or t.numel() == 0:
        return False
    span = t.numel() if t.is_contiguous() else 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return first + span * t.element_size() > start


def _describe(x, gate, mask, B, L, D, form):
    (xb, xs, _), (gb, gs, _) = x.stride(), gate.stride()
    return nat.GatedScanDesc(xb, xs, gb, gs, 0 if mask is None else mask.stride(0), B, L, D, DTYPES[x.dtype],
                             nat.GATED_SCAN_FORMS[form])


def _forward(x, gate, mask, state, last, form, train):
    """(out, last, the residual of a training call, the descriptor, the scratch's size, the addresses that it read)."""
    B, L, D = x.shape
    out = x.new_empty((B, L, D))
    if last is None:
        last = x.new_empty((B, D), dtype=torch.float32)
    desc = _describe(x, gate, mask, B, L, D, form)
    lib = nat.load()
    residual = _scratch(x, lib.ews_gated_scan_residual_bytes(desc)) if train else None
    size = lib.ews_gated_scan_workspace_bytes(desc)
    ws = _scratch(x, size)
    at = x.data_ptr(), gate.data_ptr(), _ptr(mask)
    nat.check(launch(x.device, lib.ews_gated_scan_forward, desc, *at, _ptr(state), out.data_ptr(), last.data_ptr(),
                     _ptr(residual), _ptr(ws)), "ews_gated_scan_forward")
    return out, last, residual, desc, size, at


def _come_back(x, gate, mask, residual, desc, dtype, dev):
    """Saved tensors that are not where the forward left them, as the library can read them."""
    shape = desc.batch, desc.length, desc.dim
    size = nat.load().ews_gated_scan_residual_bytes(desc)
    if returned(mask, torch.bool, shape[:2], dev) is not None:
        mask = mask.contiguous()
    x, gate = _neighbours(returned(x, dtype, shape, dev)), _neighbours(returned(gate, dtype, shape, dev))
    return x, gate, mask, aligned(returned(residual, torch.uint8, (size,), dev))


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, mask, form):
        out, last, residual, desc, size, at = _forward(x, gate, mask, state, None, form, True)
        ctx.save_for_backward(x, gate, mask, residual)
        ctx.args = desc, size, form, at, (residual.data_ptr(), x.stride(), gate.stride(),
                                            mask is not None and mask.stride(), x.dtype)
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once
    def backward(ctx, gout, glast):
        if gout is None and glast is None:
            return None, None, None, None, None
        x, gate, mask, residual = ctx.saved_tensors
        desc, size, form, forward_at, (left, x_strides, gate_strides, mask_strides, dtype) = ctx.args
        at, starts = (x.data_ptr(), gate.data_ptr(), _ptr(mask)), residual.data_ptr()
        if (at != forward_at or starts != left or x.stride() != x_strides or gate.stride() != gate_strides
                or (mask_strides and mask.stride() != mask_strides) or x.dtype is not dtype or gate.dtype is not dtype):
            x, gate, mask, residual = _come_back(x, gate, mask, residual, desc, dtype,
                                                 (glast if gout is None else gout).device)
            desc = _describe(x, gate, mask, *x.shape, form)  # the residual's and the scratch's sizes ask for no strides
            at, starts = (x.data_ptr(), gate.data_ptr(), _ptr(mask)), residual.data_ptr()
        if gout is not None:
            gout = gout.contiguous()
        if glast is not None:
            glast = glast.contiguous()
        gx, ggate = x.new_empty(x.shape), x.new_empty(x.shape)
        gstate = x.new_empty((x.shape[0], x.shape[2]), dtype=torch.float32) if ctx.needs_input_grad[2] else None
        lib = nat.load()
        ws = _scratch(x, size)
        nat.check(launch(x.device, lib.ews_gated_scan_backward, desc, *at, starts, _ptr(gout), _ptr(glast),
                         gx.data_ptr(), ggate.data_ptr(), _ptr(gstate), _ptr(ws)), "ews_gated_scan_backward")
        return gx, ggate, gstate, None, None


def gated_scan(x, gate, state=None, mask=None, form="convex", last=None):
    """The states ``h`` (B, L, D) of a recurrence with a gate for every step and channel, and the last one (B, D)::

        convex   h_t = a_t h_{t-1} + (1 - a_t) x_t    a_t = sigmoid(gate_t)
        linear   h_t = gate_t h_{t-1} + x_t

    x and gate (B, L, D), both float32 or both bfloat16 on the HIP device; any strides, read where they are if a
    step's channels are neighbours (the halves of a joint projection). ``h`` is of their type; states are summed in
    float32 and the last one is handed back in float32, unrounded. ``state`` (B, D) float32 is the state before the
    first step (default zero). ``mask`` (B, L) or (L,) bool: a step off it leaves the state as it is, whatever x and
    gate hold there (NaN too). Differentiable in x, gate and state (reverse mode). Steps are composed over stretches
    of a sequence: where a stretch's product of linear gates leaves float32's range, its states are infinite or NaN,
    also where they would have been zero.

    One token at a time is L = 1. ``last`` (B, D) float32, contiguous, takes the last state, and may be ``state``
    itself: a decoding loop that updates its state in place, also in a captured graph. It is for calls that record no
    gradients."""
    if form not in nat.GATED_SCAN_FORMS:
        raise ValueError(f"form must be one of {tuple(nat.GATED_SCAN_FORMS)}, got {form!r}")
    if x.dim() != 3 or x.shape[2] == 0:
        raise ValueError(f"x must be (B, L, D) with D >= 1, got {tuple(x.shape)}")
    if gate.shape != x.shape:
        raise ValueError(f"gate must be {tuple(x.shape)}, got {tuple(gate.shape)}")
    B, L, D = x.shape
    check_tensor("x", x)
    if gate.dtype is not x.dtype:
        raise TypeError(f"gate is {gate.dtype}, x {x.dtype}")
    if mask is not None:
        if mask.dtype is not torch.bool:
            raise TypeError(f"mask must be bool, got {mask.dtype}")
        if mask.shape != (B, L) and mask.shape != (L,):
            raise ValueError(f"mask must be {(B, L)} or {(L,)}, got {tuple(mask.shape)}")
    for name, t in (("state", state), ("last", last)):
        if t is None:
            continue
        if t.dtype is not torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        if t.shape != (B, D):
            raise ValueError(f"{name} must be {(B, D)}, got {tuple(t.shape)}")
    for name, t in (("gate", gate), ("mask", mask), ("state", state), ("last", last)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    refuse_tangents((x, gate, state, last))
    train = torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                         (state is not None and state.requires_grad))
    if last is not None:
        if train:
            raise ValueError("last is written in place: call under torch.no_grad(), or take the state that is returned")
        if not last.is_contiguous():
            raise ValueError("last must be contiguous")
        start = last.data_ptr()
        end = start + last.numel() * 4
        own = state is None or state is last or (state.data_ptr() == start and state.is_contiguous())
        if _touches(x, start, end) or _touches(gate, start, end) or not own and _touches(state, start, end):
            raise ValueError("last overlaps x, gate or a part of state: it may be state itself or apart from them all")
    if B == 0 or L == 0:  # no step: the state stays
        end = x.new_zeros((B, D), dtype=torch.float32) if state is None else state.clone()
        return x * gate, end if last is None else last.copy_(end)
    x, gate = _neighbours(x), _neighbours(gate)
    if mask is not None:
        mask = mask.expand(B, L)
        if mask.stride(1) != 1 and L > 1:
            mask = mask.contiguous()
    if state is not None:
        state = state.contiguous()
    if train:
        return _GatedScan.apply(x, gate, state, mask, form)
    given = last is not None
    out, last, *_ = _forward(x, gate, mask, state, last, form, False)
    if given:
        increment_version(last)  # a graph that has saved it refuses its backward, as after torch's own writes
    return out, last
