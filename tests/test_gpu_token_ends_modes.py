"""How the token model's ends stand with torch's other ways to differentiate: a derivative that is not formed is refused,
never dropped."""

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
