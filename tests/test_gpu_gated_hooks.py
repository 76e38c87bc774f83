"""Gradients where hooks on saved tensors bring them back contiguous, or off their 16-byte addresses: those without."""

import contextlib

import pytest
import torch
import torch.utils.checkpoint

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def _off(t, by=1):
    """t's numbers contiguous, ``by`` elements behind a 16-byte address."""
    size = t.element_size()
    flat = torch.empty(t.numel() * size + 64, dtype=torch.uint8, device=t.device)[by * size:][:t.numel() * size]
    return flat.view(t.dtype).view(t.shape).copy_(t)


def _hooks(kind):
    hooks = torch.autograd.graph.saved_tensors_hooks
    return {"none": contextlib.nullcontext, "cpu": torch.autograd.graph.save_on_cpu,
            "contiguous": lambda: hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
            "off": lambda: hooks(_off, lambda t: t)}[kind]()


@pytest.mark.parametrize("kind", ["cpu", "contiguous", "off"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,D", [(2, 300, 24), (2, 9, 25), (1, 2100, 24), (600, 20, 450)])
def test_scan_of_halves(B, L, D, dtype, kind):
    """The halves of a joint projection, a mask for all sequences: strips, threads alone, segments."""
    print(f"{B} {L} {D} {dtype} {kind}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(B + L + D)
    joint = torch.randn(B, L, 2 * D, generator=g, device="cuda").to(dtype).requires_grad_()
    state = torch.randn(B, D, generator=g, device="cuda", requires_grad=True)
    up = torch.randn(B, L, D, generator=g, device="cuda").to(dtype)
    mask = torch.arange(L, device="cuda") % 5 != 0
    grads = []
    for k in ("none", kind):
        with _hooks(k):
            h, last = E.gated_scan(*joint.chunk(2, -1), state=state, mask=mask)
        grads.append(torch.autograd.grad((h, last), (joint, state), (up, torch.ones_like(last))))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoints(dtype, reentrant):
    """Both operators formed again in the backward, between operations whose results are formed again too."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 300, 72, generator=g, device="cuda").to(dtype).requires_grad_()
    w, o = ((0.2 * torch.randn(n, 72, generator=g, device="cuda")).to(dtype).requires_grad_() for n in (144, 200))

    def block(t):
        h, last = E.gated_scan(*torch.nn.functional.linear(t, w).chunk(2, -1))
        return E.gated_linear(h, o, activation="silu"), last

    up = torch.randn(2, 300, 100, generator=g, device="cuda").to(dtype)
    grads = []
    for call in (block, lambda t: torch.utils.checkpoint.checkpoint(block, t, use_reentrant=reentrant)):
        for p in (x, w, o):
            p.grad = None
        y, last = call(x)
        torch.autograd.backward((y, last), (up, torch.ones_like(last)))
        grads.append([p.grad for p in (x, w, o)])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["cpu", "contiguous", "off"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", [(7, 128, 96), (200, 128, 96), (200, 64, 40), (300, 136, 130), (9, 1030, 70)])
def test_linear_of_rows_apart(N, H, F, dtype, kind):
    """Rows of x and of the weights apart: few rows, tiles, narrow maps, widths that have to be packed. Sums are of the
    same numbers in the same order, whether the rows are packed or read as they are."""
    print(f"{N} {H} {F} {dtype} {kind}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(N + H + F)

    def apart(rows, cols, by):
        wide = torch.randn(rows, cols + by, generator=g, device="cuda").to(dtype).requires_grad_()
        return wide, wide[:, :cols]

    for joint in (True, False):
        leaves, views = zip(apart(N, H, 8), apart(2 * F if joint else F, H, 16), *([] if joint else [apart(F, H, 16)]))
        up = torch.randn(N, F, generator=g, device="cuda").to(dtype)
        grads = []
        for k in ("none", kind):
            with _hooks(k):
                y = E.gated_linear(views[0], views[1], None, *views[2:], activation="silu")
            grads.append(torch.autograd.grad(y, leaves, up))
        for a, b in zip(*grads):
            assert torch.equal(a, b)
