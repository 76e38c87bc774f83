"""Gradient clipping by the global norm over many tensors (csrc/ews_clip.hip): the end of a training step (the
reference's optax.clip_by_global_norm in its trainers' optimisers)."""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.graph import increment_version

from . import _native as nat
from .embed import DTYPES, check_tensor, launch, refuse_tangents


def _dense(t):
    """Whether t's elements fill one stretch of memory, each once, in whatever order."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _by_place(tensors):
    """The tensors by the memory that they name; several of the same (one named twice, two views alike) give one. Empty
    ones name none."""
    places = {}
    for t in tensors:
        n = t.numel()
        places[(t.data_ptr(), n, None if t.is_contiguous() else (t.shape, t.stride())) if n else id(t)] = t
    return places


def _check(tensors):
    dev = tensors[0].device
    for t in tensors:
        if t.dtype in DTYPES and t.device == dev and t.layout is torch.strided and t.is_cuda:
            continue
        if t.layout is not torch.strided:
            raise TypeError(f"gradients must be dense tensors, got layout {t.layout}")
        check_tensor("every gradient", t)
        raise ValueError(f"gradients are on {dev} and {t.device}")
    refuse_tangents(tensors)


def _norm_and_scale(tensors, outs, max_norm):
    """The norm of tensors; where outs is not None, outs = the clipped tensors (outs is tensors: in place, memory that
    is named twice counting once)."""
    lib = nat.load()
    dev = tensors[0].device
    src = dst = tensors
    if not all([t.is_contiguous() for t in tensors]):
        src = dst = [t if _dense(t) else t.contiguous() for t in tensors]
    if outs is not None and outs is not tensors:
        dst = outs
        if src is not tensors or not all([o.is_contiguous() for o in outs]):
            dst = [o if _dense(o) and o.stride() == s.stride() else torch.empty_like(s) for o, s in zip(outs, src)]
    n, at = len(src), [t.data_ptr() for t in src]
    to = at if outs is None or dst is src else [t.data_ptr() for t in dst]
    if outs is not None and len(set(to if dst is outs else [t.data_ptr() for t in outs])) < n:
        places = _by_place(outs)
        if len(places) < n:  # in place, two workgroups would scale it once or twice, as it happens
            if outs is not tensors:
                raise ValueError("out names the same memory twice")
            once = list(places.values())
            return _norm_and_scale(once, once, max_norm)
    ptrs, counts = (ctypes.c_uint64 * n)(*at), (ctypes.c_int64 * n)(*[t.numel() for t in src])
    out = ptrs if to is at else (ctypes.c_uint64 * n)(*to)
    types = (ctypes.c_int32 * n)(*[DTYPES[t.dtype] for t in src])
    result = torch.empty(2, device=dev, dtype=torch.float32)
    ws = torch.empty(int(lib.ews_clip_workspace_bytes(n, counts)), device=dev, dtype=torch.uint8)
    nat.check(launch(dev, lib.ews_clip, n, ptrs, out, counts, types, max_norm, 0 if outs is None else 1,
                     result.data_ptr(), ws.data_ptr()), "ews_clip")
    if outs is not None:
        increment_version(outs)  # a graph that has saved one of them refuses its backward, as after torch's own writes
        if dst is not outs:
            for o, d in zip(outs, dst):
                if o is not d:
                    o.copy_(d)
    return result[0]


def _max_norm(max_norm):
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


@torch.no_grad()
def global_grad_norm(tensors):
    """The square root of the sum of all squares over float32 and bfloat16 tensors of any shapes and strides on one HIP
    device, a float32 number there; squares are added in float64. No tensors: 0 on the CPU."""
    tensors = list(tensors)
    if not tensors:
        return torch.zeros(())
    _check(tensors)
    return _norm_and_scale(tensors, None, 0.0)


@torch.no_grad()
def clip_grads(grads, max_norm, out=None):
    """(norm, clipped): ``grads`` times ``min(1, max_norm / (norm + 1e-6))``, written to the tensors of ``out`` (same
    shapes and types; a tensor of grads itself: in place; otherwise without overlap, and no two of the same memory) or
    to new ones."""
    grads = list(grads)
    max_norm = _max_norm(max_norm)
    if not grads:
        return torch.zeros(()), []
    _check(grads)
    if out is None:
        out = [torch.empty_like(t) for t in grads]
    else:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out has {len(out)} tensors for {len(grads)} gradients")
        _check(out)
        for g, o in zip(grads, out):
            if g.shape != o.shape or g.dtype is not o.dtype or g.device != o.device:
                raise ValueError(f"out has {o.dtype} {tuple(o.shape)} on {o.device} for {g.dtype} {tuple(g.shape)} on "
                                 f"{g.device}")
    return _norm_and_scale(grads, out, max_norm), out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """Scales the gradients of ``parameters`` (an iterable, or one) in place by ``min(1, max_norm / (norm + 1e-6))`` and
    returns their norm, a float32 number on the device; the host does not wait. Parameters without a gradient are left
    out; one that is named twice, or whose gradient is another's memory, counts once. A norm that is not finite scales
    by 0 (infinite) or NaN, as the formula does."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = list(dict.fromkeys(p.grad for p in parameters if p.grad is not None))
    max_norm = _max_norm(max_norm)
    if not grads:
        return torch.zeros(())
    _check(grads)
    return _norm_and_scale(grads, grads, max_norm)
