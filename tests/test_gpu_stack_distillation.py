"""``StackedEWS.distillation_loss`` against a distillation in float64 of the model's own logits: the same float32 blocks on
both sides, so the loss may differ by the rounding of a float32 loss (1e-5 of its size); gradients as in the cross entropy's
test: the stack's bar (1e-4, max|a-b| / max|b|) and four times what torch's float32 head itself is off."""

import pytest
import torch
from torch.nn.utils import parametrize

import ews_mi355x as E
from ews_mi355x.loss import logits_distillation

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _model(label_dim, **kw):
    g = torch.Generator().manual_seed(1)
    blocks = [dict(a_param=E.AParamEFM(torch.randn(8, generator=g))) for _ in range(2)]
    return E.StackedEWS(2, 11, 16, label_dim, per_block_kwargs=blocks,
                        block_kwargs=dict(m=8, n=2, leaf="series", series_q=8, channel_stage="glu", dropout_rate=0.0),
                        key=2, **kw).to(DEV)


def _teacher(shape, V, K, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    index = torch.rand(*shape, V, generator=g, device=DEV).argsort(-1)[..., :K].clone()
    index[torch.rand(*shape, K, generator=g, device=DEV) < 0.2] = -1
    return index, 2.0 * torch.randn(*shape, K, generator=g, device=DEV)


def _double(z, index, t, T):
    """Rows' losses and which have an entry, in float64."""
    has = index >= 0
    teacher = (t.double() / T).masked_fill(~has, -float("inf"))
    teacher = torch.where(has.any(-1, keepdim=True), teacher, 0.0)
    logp = torch.log_softmax(teacher, -1)
    logq = torch.log_softmax(z.double() / T, -1).gather(-1, index.clamp(min=0))
    each = torch.where(has, logp.exp() * (logp.masked_fill(~has, 0.0) - logq), 0.0)
    return T * T * each.sum(-1), has.any(-1)


def _logits(model, h, dtype):
    heads = model.head if isinstance(model.head, torch.nn.ModuleList) else [model.head]
    out = []
    for head in heads:
        x, w = h.to(dtype), head.weight.to(dtype)
        if model.cosine_head_tau is None:
            out.append(x @ w.t() + head.bias.to(dtype))
        else:
            x = x / (x.norm(dim=-1, keepdim=True) + 1e-8)
            out.append(x @ (w / (w.norm(dim=1, keepdim=True) + 1e-8)).t() / model.cosine_head_tau)
    return out


@pytest.mark.parametrize("tau,heads,mode", [(None, (9,), "seq2seq"), (0.2, (9,), "seq2seq"), (None, (9, 13), "seq2seq"),
                                            (None, (9, 13), "mean_pool")])
def test_against_the_models_own_logits(tau, heads, mode):
    T = 2.0
    model = _model(heads if len(heads) > 1 else heads[0], cosine_head_tau=tau, head_mode=mode)
    X = torch.randint(1, 11, (3, 20), device=DEV)
    mask = torch.arange(20, device=DEV)[None] < torch.tensor([[20], [13], [7]], device=DEV)
    shape = (3, 20) if mode == "seq2seq" else (3,)
    teachers = [_teacher(shape, V, 5, V) for V in heads]
    params = list(model.parameters())

    def reference(dtype):
        h = model.hidden(X, mask=mask)
        if mode == "mean_pool":
            h = model._pool(h, mask)
        total = 0.0
        for z, (index, t) in zip(_logits(model, h, dtype), teachers):
            if mode == "seq2seq":
                index = index.masked_fill(~mask[..., None], -1)
            rows, kept = _double(z, index, t, T)
            total = total + rows.sum() / kept.sum()
        return total

    indices, logits = (tuple(v) if len(heads) > 1 else v[0] for v in zip(*teachers))
    loss = model.distillation_loss(X, indices, logits, temperature=T, mask=mask)
    want, plain = reference(torch.float64), reference(torch.float32)
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    got, exact, near = (torch.autograd.grad(v, params, allow_unused=True) for v in (loss, want, plain))
    for (name, _), a, r, b in zip(model.named_parameters(), got, exact, near):
        assert (a is None) == (r is None), name
        if a is not None:
            own, theirs = float((a - r).abs().max()), float((b - r).abs().max())
            assert own <= 1e-4 * float(r.abs().max()) + 4.0 * theirs, (name, own, theirs)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_a_called_head_answers_as_the_fused_one(reduction):
    """A head that is more than a linear map is called as the module it is."""
    model = _model(9)
    X = torch.randint(1, 11, (3, 20), device=DEV)
    index, t = _teacher((3, 20), 9, 4)
    want = model.distillation_loss(X, index, t, temperature=1.5, reduction=reduction)
    calls = []
    handle = model.head.register_forward_hook(lambda *a: calls.append(1))
    got = model.distillation_loss(X, index, t, temperature=1.5, reduction=reduction)
    handle.remove()
    assert calls and got.shape == want.shape
    # both are float32 losses of logits of a few units, 60 rows: 2^-18 a row is some thirty roundings
    assert float((got - want).detach().abs().max()) <= 2.0**-18 * (60 if reduction == "sum" else 1) * 4

    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    parametrize.register_parametrization(model.head, "weight", Twice())
    h = model.hidden(X)
    z = model.head(h)
    ref = logits_distillation(z, index, t, 1.5, reduction)
    got = model.distillation_loss(X, index, t, temperature=1.5, reduction=reduction)
    assert float((got - ref).detach().abs().max()) <= 2.0**-18 * (60 if reduction == "sum" else 1) * 4


def test_refusals():
    model = _model((9, 13))
    X = torch.randint(1, 11, (3, 20), device=DEV)
    index, t = _teacher((3, 20), 9, 4)
    with pytest.raises(ValueError, match="2 head"):
        model.distillation_loss(X, index, t)
    with pytest.raises(ValueError, match="batch"):
        model.distillation_loss(X[0], (index, index), (t, t))
    with pytest.raises(ValueError, match="indices must be"):
        model.distillation_loss(X, (index[:, 1:], index), (t, t))
