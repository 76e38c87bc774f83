"""``StackedEWS.loss`` (embedding lookup, blocks, linear cross entropy) against a cross entropy of the model's own
logits. Both run the same float32 blocks, so the loss may differ by the rounding of a float32 cross entropy (1e-5 of its
size). The gradients are compared with those through a float64 head on the same hidden rows: the blocks' backward is the
same linear map of the head's cotangent in all, but may amplify its last bits (an input of these cases does so a
thousandfold), so the yardstick beside the stack's bar (1e-4, max|a-b| / max|b|) is how far torch's float32 head itself
is from the float64 one, four times. And the example that trains with it and with clipping."""

import math
import os
import sys

import pytest
import torch
import torch.nn.functional as F

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _model(label_dim, tokens=True, **kw):
    g = torch.Generator().manual_seed(1)
    blocks = [dict(a_param=E.AParamEFM(torch.randn(8, generator=g))) for _ in range(2)]
    return E.StackedEWS(2, 11 if tokens else 3, 16, label_dim, tokens=tokens, per_block_kwargs=blocks,
                        block_kwargs=dict(m=8, n=2, leaf="series", series_q=8, channel_stage="glu", dropout_rate=0.0),
                        key=2, **kw).to(DEV)


def _logits64(model, X, mask):
    """The model's logits by a float64 head on its float32 hidden rows."""
    h = model.hidden(X, mask=mask)
    if model.head_mode == "mean_pool":
        h = model._pool(h, mask)
    heads = model.head if isinstance(model.head, torch.nn.ModuleList) else [model.head]
    out = []
    for head in heads:
        x, w = h.double(), head.weight.double()
        if model.cosine_head_tau is None:
            out.append(x @ w.t() + head.bias.double())
        else:
            x = x / (x.norm(dim=-1, keepdim=True) + 1e-8)
            out.append(x @ (w / (w.norm(dim=1, keepdim=True) + 1e-8)).t() / model.cosine_head_tau)
    return tuple(out) if len(out) > 1 else out[0]


def _compare(model, X, targets, mask, reference, **kw):
    params = list(model.parameters())

    def grads(loss):
        return torch.autograd.grad(loss, params, allow_unused=True)

    loss = model.loss(X, targets, mask=mask, **kw)
    ref = reference(model(X, mask=mask))
    assert abs(float(loss.detach()) - float(ref.detach())) <= 1e-5 * abs(float(ref.detach()))
    exact = grads(reference(_logits64(model, X, mask)))
    for (name, _), a, b, r in zip(model.named_parameters(), grads(loss), grads(ref), exact):
        assert (a is None) == (r is None), name
        if a is not None:
            own, plain = float((a - r).abs().max()), float((b - r).abs().max())
            assert own <= 1e-4 * float(r.abs().max()) + 4.0 * plain, (name, own, plain)


@pytest.mark.parametrize("tau", [None, 0.2])
def test_positions(tau):
    g = torch.Generator().manual_seed(0)
    X = torch.randint(0, 11, (6, 40), generator=g).to(DEV)
    y = torch.randint(0, 7, (6, 40), generator=g).to(DEV)
    mask = (torch.arange(40)[None] < torch.tensor([40, 31, 1, 17, 39, 5])[:, None]).to(DEV)
    model = _model(7, cosine_head_tau=tau)
    _compare(model, X, y, mask, lambda z: F.cross_entropy(z[mask], y[mask]))
    _compare(model, X, y, None, lambda z: F.cross_entropy(z.flatten(0, 1), y.flatten(), reduction="sum"),
             reduction="sum")


def test_pooled_and_several_heads():
    g = torch.Generator().manual_seed(3)
    X = torch.randn(5, 33, 3, generator=g).to(DEV)
    ys = tuple(torch.randint(0, k, (5,), generator=g).to(DEV) for k in (4, 9))
    model = _model((4, 9), tokens=False, head_mode="mean_pool")
    _compare(model, X, ys, None, lambda z: F.cross_entropy(z[0], ys[0]) + F.cross_entropy(z[1], ys[1]))
    with pytest.raises(ValueError, match="head"):
        model.loss(X, ys[0])
    with pytest.raises(ValueError, match="batch"):
        model.loss(X[0], ys)


def test_example_learns():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import train_tokens
    finally:
        sys.path.pop(0)
    norms = []
    losses = train_tokens.train(steps=60, report=lambda step, loss, norm: norms.append(norm))
    assert bool(torch.isfinite(losses).all()) and bool(torch.isfinite(torch.stack(norms)).all())
    assert abs(float(losses[0]) - math.log(16.0)) < 1.0
    assert float(losses[-10:].mean()) < 0.95 * float(losses[:10].mean())
