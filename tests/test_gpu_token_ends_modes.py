"""How the token model's ends stand with torch's other ways to differentiate: a derivative that is not formed is
refused, never dropped."""

import pytest
import torch
from torch.autograd import forward_ad

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _calls(dual):
    """Every operator with one of its operands carrying a tangent."""
    t = torch.tensor([1, 0, 2], device=DEV)
    w, h, b = torch.randn(5, 8, device=DEV), torch.randn(3, 8, device=DEV), torch.randn(5, device=DEV)
    yield "lookup, weight", lambda: E.embedding_lookup(t, dual(w))
    for reduction in ("mean", "none"):
        yield "loss, hidden", lambda: E.linear_cross_entropy(dual(h), w, t, bias=b, reduction=reduction)
        yield "loss, weight", lambda: E.linear_cross_entropy(h, dual(w), t, reduction=reduction)
        yield "loss, bias", lambda: E.linear_cross_entropy(h, w, t, bias=dual(b), reduction=reduction)
    yield "norm", lambda: E.global_grad_norm([h, dual(w)])
    yield "clip", lambda: E.clip_grads([h, dual(w)], 1.0)


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(no_grad):
    with forward_ad.dual_level():
        for name, call in _calls(lambda x: forward_ad.make_dual(x, torch.ones_like(x))):
            print(name, flush=True)
            with torch.set_grad_enabled(not no_grad), pytest.raises(NotImplementedError):
                call()
        for _, call in _calls(lambda x: x):  # without tangents all is as ever
            call()


def test_jvp_is_refused():
    t = torch.tensor([1, 0, 2], device=DEV)
    w, h = torch.randn(5, 8, device=DEV), torch.randn(3, 8, device=DEV)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda x: E.embedding_lookup(t, x), (w,), (w,))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda x: E.linear_cross_entropy(x, w, t), (h,), (h,))


@pytest.mark.parametrize("strided", [False, True])
def test_clipping_in_place_is_seen_by_graphs_that_saved_the_gradient(strided):
    """A product has saved the gradient; once it is clipped the product's backward would be another number's."""

    def tensor():
        return torch.randn(8, 6, device=DEV)[:, ::2] if strided else torch.randn(8, 3, device=DEV)

    def saved(g):
        w = torch.ones(g.shape, device=DEV, requires_grad=True)
        return (w * g).sum()

    g = tensor()
    for call in (lambda: E.clip_grads([g], 1e-3, out=[g]), lambda: E.clip_grads([tensor()], 1e-3, out=[g]),
                 lambda: E.clip_grads([g], 1e6, out=[g])):
        y, before = saved(g), g._version
        call()
        assert g._version > before
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    p = torch.zeros(8, 3, device=DEV, requires_grad=True)
    p.grad = tensor()
    y = saved(p.grad)
    E.clip_grad_norm_([p], 1e-3)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    # what is only read stays as it was
    y = saved(g)
    E.global_grad_norm([g])
    E.clip_grads([g], 1e-3)
    y.backward()


def test_clipping_under_inference_mode():
    with torch.inference_mode():
        g = torch.randn(8, 3, device=DEV)
        want = g.clone()
        norm, out = E.clip_grads([g], 1e-3)
        E.clip_grads([g], 1e-3, out=[g])
        assert torch.equal(g, out[0]) and not torch.equal(g, want)


def test_memory_named_twice_is_scaled_once():
    """Two workgroups that scale one tensor in place would scale it once or twice, as it happens."""
    g = torch.randn(70, 33, device=DEV)
    p, q, r = (torch.zeros(70, 33, device=DEV, requires_grad=True) for _ in range(3))
    p.grad, q.grad = g.clone(), torch.randn(70, 33, device=DEV)
    r.grad = p.grad.view(70, 33)
    e = torch.zeros(0, device=DEV, requires_grad=True)
    e.grad = torch.zeros(0, device=DEV)
    want_norm, want = E.clip_grads([g, q.grad.clone()], 0.5)
    norm = E.clip_grad_norm_([p, q, e, r, e, p], 0.5)
    assert torch.equal(norm, want_norm)
    assert torch.equal(p.grad, want[0]) and torch.equal(q.grad, want[1])
    for out in ([g, g], [g, g.view(70, 33)]):
        with pytest.raises(ValueError, match="twice"):
            E.clip_grads([g, g], 0.5, out=out)
    none = [torch.zeros(0, device=DEV) for _ in range(2)]
    E.clip_grads(none, 0.5, out=none)
    # a row and a column that begin alike are not the same memory
    base = torch.randn(33, 40, device=DEV)
    rows = [base[:, :20], base[:, 20:]]
    assert len(E.clip_grads(rows, 0.5, out=rows)[1]) == 2
    s, t = (torch.zeros(40, device=DEV, requires_grad=True) for _ in range(2))
    line = torch.randn(80, device=DEV)
    line[0] = 0.0
    s.grad, t.grad = line[:40], line[::2]
    assert float(E.clip_grad_norm_([s, t], 1e9)) == pytest.approx(
        float((line[:40].square().sum() + line[::2].square().sum()).sqrt()), rel=1e-6)
