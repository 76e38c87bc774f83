"""Gradients of ``gated_linear`` where its operands are views: rows apart, off their 16-byte addresses, turned, V and G
at different strides. The leaves are what the views are taken of, so the layouts reach the backward; values and bounds
are those of ``test_gpu_gated_linear``."""

import pytest
import torch

import ews_mi355x as E
from test_gpu_gated_linear import DEV, DTYPES, _close, _inputs, _reference

pytestmark = pytest.mark.gpu


def _plain(t):
    leaf = t.detach().clone().requires_grad_()
    return leaf, leaf


def _apart(by):
    def make(t):
        wide = torch.full((t.shape[0], t.shape[1] + by), 7.0, device=DEV, dtype=t.dtype)
        wide[:, :t.shape[1]] = t
        leaf = wide.requires_grad_()
        return leaf, leaf[:, :t.shape[1]]

    return make


def _off(t):
    leaf = torch.cat([t.new_zeros(1), t.flatten()]).requires_grad_()
    return leaf, leaf[1:].view(t.shape)


def _turned(t):
    leaf = t.t().contiguous().requires_grad_()
    return leaf, leaf.t()


def _of_view(make, grad, shape):
    """The gradient of the view's numbers, from the leaf's."""
    if make is _off:
        return grad[1:].view(shape)
    return grad.t() if make is _turned else grad[:, :shape[1]]


LAYOUTS = [(_apart(8), _apart(16), _apart(16)), (_plain, _apart(16), _plain), (_plain, _apart(3), _plain),
           (_off, _plain, _plain), (_plain, _off, _plain), (_plain, _plain, _off), (_apart(1), _off, _off),
           (_turned, _turned, _plain), (_apart(8), _plain, _plain)]


@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", [(5, 128, 96), (50, 128, 96), (200, 128, 96), (200, 64, 48), (1100, 520, 3330)])
def test_gradients_of_views(N, H, F, dtype, layout):
    print(f"{N} {H} {F} {dtype} {layout}", flush=True)
    x, w, b, gw, gb, up = _inputs(N, H, F, dtype, joint=False)
    want = _reference(x, w, b, gw, gb, up, "silu")
    makes = LAYOUTS[layout]
    leaves, views = zip(*(m(t) for m, t in zip(makes, (x, w, gw))))
    y = E.gated_linear(views[0], views[1], b, views[2], gb, activation="silu")
    _close(y.detach(), want["y"], "y")
    for key, make, view, grad in zip("xVG", makes, views, torch.autograd.grad(y, leaves, up)):
        _close(_of_view(make, grad, view.shape), want[key], key)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [5, 200])
def test_gradients_of_a_joint_weight_of_rows_apart(N, dtype):
    x, w, b, _, _, up = _inputs(N, 128, 96, dtype)
    want = _reference(x, w, b, None, None, up, "gelu")
    for make in (_apart(16), _apart(3), _off, _turned):
        leaf, view = make(w)
        grad, = torch.autograd.grad(E.gated_linear(x, view, b, activation="gelu"), leaf, up)
        _close(_of_view(make, grad, w.shape), tuple(torch.cat(t) for t in zip(want["V"], want["G"])), "weight")


@pytest.mark.parametrize("dtype", DTYPES)
def test_upstream_gradients_of_any_layout(dtype):
    x, w, b, gw, gb, up = _inputs(200, 128, 96, dtype, joint=False)
    want = _reference(x, w, b, gw, gb, up, "relu")
    for make in (_apart(8), _off, _turned):
        x1 = x.clone().requires_grad_()
        grad, = torch.autograd.grad(E.gated_linear(x1, w, b, gw, gb, activation="relu"), x1, make(up)[1].detach())
        _close(grad, want["x"], "x")
