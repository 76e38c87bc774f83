"""``StackedEWS.loss`` where the embedding or the head is more than its weights: hooks that set them (pruning, weight
normalisation), hooks that change or watch the result, modules with options of their own. The loss has to be a cross
entropy of what ``forward`` returns.

Both sides run the same float32 blocks; the head's two forms differ by a few 2^-24 of a logit of a few units (1e-5 of
the loss allowed), and the blocks' backward may amplify a cotangent's last bits a thousandfold: 8 * 2^-24 * 1000 = 5e-4
of a gradient's largest number, 1e-3 allowed."""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.utils import prune

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _model(label_dim=7, **kw):
    g = torch.Generator().manual_seed(1)
    blocks = [dict(a_param=E.AParamEFM(torch.randn(8, generator=g)))]
    return E.StackedEWS(1, 11, 16, label_dim, tokens=True, per_block_kwargs=blocks, key=2,
                        block_kwargs=dict(m=8, n=2, leaf="series", series_q=8, channel_stage="glu", dropout_rate=0.0),
                        **kw).to(DEV)


def _data():
    g = torch.Generator().manual_seed(0)
    X = torch.randint(0, 11, (6, 40), generator=g).to(DEV)
    y = torch.randint(0, 7, (6, 40), generator=g).to(DEV)
    mask = (torch.arange(40)[None] < torch.tensor([40, 31, 1, 17, 39, 5])[:, None]).to(DEV)
    return X, y, mask


def _compare(model, reduction="mean"):
    X, y, mask = _data()
    params = list(model.parameters())
    loss = model.loss(X, y, mask=mask, reduction=reduction)  # first: nothing has set the weights anew since the change
    got = torch.autograd.grad(loss, params, torch.ones_like(loss), allow_unused=True)
    rows = F.cross_entropy(model(X, mask=mask).flatten(0, 1), y.flatten(), reduction="none").view(6, 40)
    ref = rows * mask if reduction == "none" else rows[mask].mean() if reduction == "mean" else rows[mask].sum()
    want = torch.autograd.grad(ref, params, torch.ones_like(ref), allow_unused=True)
    assert loss.shape == ref.shape
    loss, ref = loss.detach(), ref.detach()
    assert float((loss - ref).abs().max()) <= 1e-5 * float(ref.abs().max())
    for (name, _), a, b in zip(model.named_parameters(), got, want):
        assert (a is None) == (b is None), name
        if a is not None:
            assert float((a - b).abs().max()) <= 1e-3 * float(b.abs().max()), name


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("which", ["head", "embedding"])
def test_pruned_weights(which, reduction):
    model = _model()
    module = getattr(model, which)
    prune.random_unstructured(module, "weight", amount=0.5)
    with torch.no_grad():
        module.weight_orig.mul_(3.0)  # an optimiser's step: the hook forms the weight from it at the next call
    _compare(model, reduction)


def test_weight_normalised_head():
    model = _model()
    with pytest.warns(FutureWarning):
        nn.utils.weight_norm(model.head)
    with torch.no_grad():
        model.head.weight_g.mul_(2.0)
    _compare(model)


def test_parametrised_head():
    model = _model()
    nn.utils.parametrizations.weight_norm(model.head)
    with torch.no_grad():
        model.head.parametrizations.weight.original0.mul_(2.0)
    _compare(model)


@pytest.mark.parametrize("which", ["head", "embedding"])
def test_hooks_run(which):
    model = _model()
    module = getattr(model, which)
    seen = []
    handles = [module.register_forward_pre_hook(lambda m, args: seen.append("pre")),
               module.register_forward_hook(lambda m, args, out: out * 2.0),
               module.register_full_backward_hook(lambda m, gin, gout: seen.append("backward"))]
    _compare(model)
    assert seen == ["pre", "backward"] * 2
    for h in handles:
        h.remove()
    _compare(model)
    assert len(seen) == 4


def test_hooks_of_all_modules_run():
    model = _model()
    seen = []
    handle = nn.modules.module.register_module_forward_hook(lambda m, args, out: seen.append(m))
    try:
        _compare(model)
    finally:
        handle.remove()
    assert seen.count(model.head) == 2 and seen.count(model.embedding) == 2


def test_modules_with_options_or_a_forward_of_their_own():
    model = _model()
    padded = nn.Embedding(11, 16, padding_idx=4).to(DEV)
    model.embedding = padded
    _compare(model)
    model.embedding = nn.Embedding(11, 16, max_norm=0.5).to(DEV)
    _compare(model)

    class Doubled(nn.Linear):
        def forward(self, x):
            return 2.0 * super().forward(x)

    model = _model()
    model.head = Doubled(16, 7).to(DEV)
    _compare(model)
    model.head = nn.Sequential(nn.Linear(16, 9), nn.Tanh(), nn.Linear(9, 7)).to(DEV)
    _compare(model)


def test_a_called_head_answers_as_the_fused_one():
    """Ignored rows, targets outside the vocabulary, no kept row, refusals."""
    model = _model()
    X, y, mask = _data()
    y[0, 3], y[1, 2] = -100, 8
    want = model.loss(X, y, mask=mask, reduction="none")
    handle = model.head.register_forward_hook(lambda m, args, out: None)
    got = model.loss(X, y, mask=mask, reduction="none")
    assert bool(torch.isnan(got[1, 2])) and int(torch.isnan(got).sum()) == 1 and not bool(got[0, 3])
    assert torch.allclose(got, want, rtol=0.0, atol=1e-5, equal_nan=True)
    assert float(model.loss(X, torch.full_like(y, -100))) == 0.0
    for call, kind in ((lambda: model.loss(X, y[:, :5]), ValueError), (lambda: model.loss(X, y.float()), TypeError),
                       (lambda: model.loss(X, y, reduction="max"), ValueError)):
        with pytest.raises(kind):
            call()
        handle.remove()
        with pytest.raises(kind):
            call()
        handle = model.head.register_forward_hook(lambda m, args, out: None)
