"""What ``linear_distillation`` refuses before any device is touched, the library's own checks, and the torch operations
for heads that are more than a linear map against the definition in float64."""

import ctypes
import math

import pytest
import torch

import ews_mi355x as E
from ews_mi355x import _native as nat
from ews_mi355x.loss import logits_distillation

BASE = dict(hidden=torch.zeros(6, 4), weight=torch.zeros(9, 4), indices=torch.zeros(6, 3, dtype=torch.long),
            logits=torch.zeros(6, 3))


@pytest.mark.parametrize("change,error,says", [
    (dict(reduction="max"), ValueError, "reduction must be"),
    (dict(weight=torch.zeros(9)), ValueError, "weight must be"),
    (dict(hidden=torch.zeros(6, 5)), ValueError, "hidden must be"),
    (dict(bias=torch.zeros(8)), ValueError, "bias must be"),
    (dict(indices=torch.zeros(6, dtype=torch.long)), ValueError, "indices must be"),
    (dict(indices=torch.zeros(5, 3, dtype=torch.long)), ValueError, "indices must be"),
    (dict(indices=torch.zeros(6, 0, dtype=torch.long), logits=torch.zeros(6, 0)), ValueError, "1 to 1024 entries"),
    (dict(indices=torch.zeros(6, 1025, dtype=torch.long), logits=torch.zeros(6, 1025)), ValueError, "1 to 1024 entries"),
    (dict(logits=torch.zeros(6, 2)), ValueError, "logits must be"),
    (dict(temperature=0.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(temperature=2e6), ValueError, "temperature"),
    (dict(indices=torch.zeros(6, 3)), TypeError, "int64 or int32"),
    (dict(logits=torch.zeros(6, 3, requires_grad=True)), ValueError, "detach"),
    (dict(), RuntimeError, "HIP device"),
])
def test_refusals(change, error, says):
    with pytest.raises(error, match=says):
        E.linear_distillation(**{**BASE, **change})


def _desc(head=None, **kw):
    base = dict(hidden_stride=4, weight_stride=4, ignore_index=0, rows=6, hidden=4, vocab=9, dtype=0, bias_dtype=0,
                reduction=1)
    base.update(head or {})
    top = dict(index_stride=3, logit_stride=3, entries=3, index_bytes=8, logit_dtype=0, temperature=1.0)
    top.update(kw)
    return nat.DistillDesc(nat.LossDesc(**base), **top)


@pytest.mark.parametrize("bad", [dict(entries=0), dict(entries=1025), dict(index_bytes=2), dict(logit_dtype=5),
                                 dict(temperature=0.0), dict(temperature=float("nan")), dict(index_stride=-1),
                                 dict(head=dict(rows=0)), dict(head=dict(dtype=9)), dict(head=dict(hidden_stride=3))])
def test_library_refuses(bad):
    lib, one = nat.load(), ctypes.c_void_p(16)
    d = _desc(**bad)
    assert lib.ews_distill_workspace_bytes_for(d, one, 1) == 0 and lib.ews_distill_keeps(d) == 0
    assert lib.ews_distill_forward(d, one, one, None, one, one, one, one, None) in (-2, -4)
    assert lib.ews_distill_train(d, one, one, None, one, one, None, one, one, one, None, one, None) in (-2, -4)
    assert lib.ews_distill_keep(d, one, one, None, one, one, one, one, one, None) in (-2, -4)
    assert lib.ews_distill_kept(d, one, one, one, one, None, one, None) in (-2, -4)


def test_library_refuses_null():
    lib, one, d = nat.load(), ctypes.c_void_p(16), _desc()
    assert lib.ews_distill_forward(None, one, one, None, one, one, one, one, None) == -1
    for hole in range(6):
        p = [one] * 6
        p[hole] = None
        assert lib.ews_distill_forward(d, p[0], p[1], None, p[2], p[3], p[4], p[5], None) == -1
    assert lib.ews_distill_train(d, one, one, None, one, one, None, one, one, one, one, one, None) == -1  # no bias


def test_scratch_of_the_entries():
    """Beside the cross entropy's: per row 12 bytes an entry, 2 every 128 tokens, and a few."""
    lib = nat.load()
    for N, V, K in ((6, 9, 3), (8192, 32000, 32), (131072, 100003, 1024)):
        d = _desc(head=dict(rows=N, vocab=V, hidden=64, hidden_stride=64, weight_stride=64, dtype=1), entries=K)
        for train in (0, 1):
            own = lib.ews_distill_workspace_bytes_for(d, 0, train)
            plain = lib.ews_loss_workspace_bytes_for(d.head, 0, train)
            assert plain < own <= plain + N * (12 * K + 2 * ((V + 255) // 128 + 2) + 16) + 2048


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_of_logits(reduction):
    g = torch.Generator().manual_seed(3)
    N, V, K, T = 30, 20, 6, 1.7
    z = torch.randn(N, V, generator=g).requires_grad_()
    index, t = torch.randint(-2, V, (N, K), generator=g), torch.randn(N, K, generator=g)
    index[4] = -1
    t[5, 2] = -math.inf
    t[6] = -math.inf
    t[index < 0] = float("nan")
    got = logits_distillation(z, index, t, T, reduction)
    zd = z.detach().double().requires_grad_()
    rows = []
    for n in range(N):
        on = [k for k in range(K) if index[n, k] >= 0 and t[n, k] != -math.inf]
        if not on:
            rows.append(zd[n].sum() * 0)
            continue
        p = torch.softmax(t[n, on].double() / T, 0)
        logq = torch.log_softmax(zd[n] / T, 0)[index[n, on]]
        rows.append(T * T * (p * (p.log() - logq)).sum())
    rows = torch.stack(rows)
    kept = sum(any(index[n, k] >= 0 and t[n, k] != -math.inf for k in range(K)) for n in range(N))
    want = rows if reduction == "none" else rows.sum() / (kept if reduction == "mean" else 1)
    # some forty float32 roundings of numbers below ten
    assert torch.allclose(got.double(), want, rtol=0, atol=40 * 10 * 2.0**-24 * (1 if reduction != "sum" else N))
    up = torch.ones_like(got)
    a, r = torch.autograd.grad(got, z, up)[0], torch.autograd.grad(want, zd, up.double())[0]
    assert torch.allclose(a.double(), r, rtol=0, atol=40 * 2.0**-23)
    index[3, 0] = V
    t[3, 0] = 0.0
    assert bool(logits_distillation(z, index, t, T, "none")[3].isnan())


@pytest.mark.parametrize("T", [32.0, 1000.0, 1e4])
def test_of_logits_at_high_temperatures(T):
    """T^2 brings out what is left of logarithms that cancel: some digits of float32, not a few of T^2 of them."""
    g = torch.Generator().manual_seed(5)
    z, t = 2 * torch.randn(12, 300, generator=g), 2 * torch.randn(12, 300, generator=g)
    index = torch.stack([torch.randperm(300, generator=g) for _ in range(12)])
    logp, logq = torch.log_softmax(t.double() / T, 1), torch.log_softmax(z.double() / T, 1).gather(1, index)
    want = T * T * (logp.exp() * (logp - logq)).sum(1)
    got = logits_distillation(z, index, t, T, "none")
    # the result's rounding, and float64's own of 300 terms of 6: T^2 2^-44
    assert bool(((got.double() - want).abs() <= 2.0**-23 * want + T * T * 2.0**-44).all())


def test_temperatures_without_digits_are_refused():
    with pytest.raises(ValueError, match="temperature must be from 1e-6 to 1e4"):
        E.linear_distillation(**{**BASE, "temperature": 2e4})
    lib, one = nat.load(), ctypes.c_void_p(16)
    d = _desc(temperature=2e4)
    assert lib.ews_distill_workspace_bytes_for(d, one, 1) == 0
    assert lib.ews_distill_forward(d, one, one, None, one, one, one, one, None) == -4
