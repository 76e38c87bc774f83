"""Embedding lookup with scaling, and its gradient by sorted tokens (csrc/ews_embed.hip): the token end of a
``StackedEWS`` (the reference's eqx.nn.Embedding, ews/block.py:473-756)."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat

DTYPES = {torch.float32: nat.DTYPE_F32, torch.bfloat16: nat.DTYPE_BF16}
_NO_PADDING = -1


def launch(dev, fn, *args):
    """fn(*args, stream) on dev's current stream, with dev the current device."""
    if dev.index == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    with torch.cuda.device(dev):
        return fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))


def once(backward):
    """``once_differentiable``, which costs a small call 5 us, where a graph of the backward is asked for; else backward
    itself."""
    refusing = once_differentiable(backward)

    def run(ctx, *grads):
        return refusing(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def returned(t, dtype, shape, dev):
    """A saved tensor (or None) as it came back: hooks on saved tensors may bring it back at another address, with other
    strides; of another type, shape or device it is refused."""
    if t is not None and (t.dtype is not dtype or t.shape != shape or t.device != dev):
        raise RuntimeError(f"a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}: it was {dtype} "
                           f"{tuple(shape)} on {dev}")
    return t


def aligned(t):
    """A saved buffer of the library's own, contiguous, at a multiple of 16 bytes (a copy only where it is not)."""
    return t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(
        memory_format=torch.contiguous_format)


def has_tangent(tensors):
    """Whether a tensor (or None) of them carries a forward-mode derivative."""
    if forward_ad._current_level < 0:  # no forward-mode differentiation is going on
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def refuse_tangents(tensors):
    """Forward-mode derivatives are not formed: a tensor (or None) that carries one is refused, as an autograd function
    without a jvp refuses it, not answered without a tangent, which would read as a derivative of zero."""
    if has_tangent(tensors):
        raise NotImplementedError("ews_mi355x has no forward-mode derivatives (jvp) of this operator")


def check_tensor(name, t):
    if not t.is_cuda:
        raise RuntimeError(f"ews_mi355x runs on a HIP device only: move {name} to the GPU (no CPU path)")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")


def row_major(t):
    """A 2-D tensor whose rows are contiguous and do not overlap (a copy only where they do), and its row stride."""
    n, w = t.shape
    if t.is_contiguous():
        return t, w
    if (t.stride(1) != 1 and w > 1) or (t.stride(0) < w and n > 1):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else w)


def _lookup(tokens, weight, scale, padding):
    """The rows, and the descriptor of the call and of its gradient."""
    shape = weight.shape
    out = weight.new_empty((*tokens.shape, shape[1]))
    n = tokens.numel()
    if n == 0:
        return out, None
    weight, stride = row_major(weight)
    desc = nat.EmbedDesc(n, stride, padding, shape[1], shape[0], DTYPES[weight.dtype], tokens.element_size(), scale)
    nat.check(launch(weight.device, nat.load().ews_embed_forward, desc, tokens.data_ptr(), weight.data_ptr(),
                     out.data_ptr()), "ews_embed_forward")
    return out, desc


class _Lookup(torch.autograd.Function):
    # A small training call costs its host time, and the backward's thread runs Python two to three times slower than
    # the caller's (each finds the interpreter's memory in the other core's cache): what the backward needs is prepared
    # in the forward, and every attribute or call spared counts.
    @staticmethod
    def forward(ctx, weight, tokens, scale, padding):
        ctx.save_for_backward(tokens)
        out, desc = _lookup(tokens, weight, scale, padding)
        ctx.args = desc, weight.shape, desc and nat.load().ews_embed_workspace_bytes(desc)
        return out

    @staticmethod
    @once
    def backward(ctx, gout):
        desc, shape, size = ctx.args
        grad = gout.new_empty(shape)
        if desc is None:
            return grad.zero_(), None, None, None
        (tokens,) = ctx.saved_tensors
        gout = gout.contiguous()
        ws = gout.new_empty(size, dtype=torch.uint8) if size else None
        nat.check(launch(gout.device, nat.load().ews_embed_backward, desc, tokens.data_ptr(), gout.data_ptr(),
                         grad.data_ptr(), ws.data_ptr() if size else None), "ews_embed_backward")
        return grad, None, None, None


def embedding_lookup(tokens, weight, scale=1.0, padding_idx=None):
    """``scale * weight[tokens]``: tokens of any shape (int64 or int32), weight (V, H) float32 or bfloat16 on the HIP
    device -> (*tokens.shape, H) in weight's type. Differentiable in weight (reverse mode): a token's gradient rows are
    added in the order of the tokens, in float32 and without atomics, so the same inputs give the same gradient bits;
    the rows of ``padding_idx`` get none. A token outside [0, V) gives a row of NaN and has no gradient (the host does
    not wait to look at the tokens)."""
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (V, H) with V, H >= 1, got {tuple(weight.shape)}")
    check_tensor("weight", weight)
    refuse_tangents((weight,))
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    if tokens.device != weight.device:
        raise ValueError(f"tokens are on {tokens.device}, weight on {weight.device}")
    padding = _NO_PADDING
    if padding_idx is not None:
        padding = int(padding_idx) + (weight.shape[0] if padding_idx < 0 else 0)
        if not 0 <= padding < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} is outside a vocabulary of {weight.shape[0]}")
    tokens = tokens.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        return _Lookup.apply(weight, tokens, float(scale), padding)
    return _lookup(tokens, weight, float(scale), padding)[0]
