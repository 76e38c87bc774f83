"""``linear_distillation`` at high temperatures and where student and teacher are alike, against float64.

With r the relative error of p / q, ep + e of ``test_gpu_linear_distillation`` (of a logit's error over T, and some
twenty roundings), a row whose entries name all tokens is T^2 sum_k q_k f(x_k) with x = p / q - 1, f'(x) = log (1 + x) =
d and f'' = 1 / (1 + x): off by T^2 sum_k q_k (|d_k| r + r^2) and (K + 32) u of itself. Other rows have 1 - sum_k q_k
too, off by e + (K + 8) u at most, times T^2."""

import math

import pytest
import torch

import ews_mi355x as E
from ews_mi355x.loss import logits_distillation

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24


def _case(N, H, V, K, dtype, spread, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + N + 7 * V + K)
    h = torch.randn(N, H, generator=g, device=DEV).to(dtype)
    w = (spread * torch.randn(V, H, generator=g, device=DEV) / math.sqrt(H)).to(dtype)
    index = torch.stack([torch.randperm(V, generator=g, device=DEV)[:K] for _ in range(N)])
    z = h.double() @ w.double().t()
    return h, w, z, index, g


def _expected(h, w, z, index, t, T):
    """Rows, their bounds, and dz, in float64."""
    (V, H), K = w.shape, index.shape[1]
    logp, logq = torch.log_softmax(t.double() / T, 1), torch.log_softmax(z / T, 1)
    lq = logq.gather(1, index)
    p, q, d = logp.exp(), lq.exp(), logp - lq
    rows = T * T * (p * d).sum(1)
    zerr = (H + 8) * U * (h.double().abs() @ w.double().abs().t()).amax(1) / T
    e = 2 * zerr + 16 * U + 2 * U * z.abs().amax(1) / T
    far = (t.double().amax(1, keepdim=True) - t.double()) / T
    r = (3 * far + K + 16) * U + e[:, None]
    bound = T * T * (torch.maximum(p, q) * (d.abs() * r + r * r)).sum(1) + (K + 32) * U * rows.abs()
    if K < V:
        bound += T * T * (e + (K + 8) * U)
    dz = logq.exp().scatter_add(1, index, -p) * T
    return rows, bound, dz


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1.0, 32.0, 100.0, 1000.0, 1e4])
@pytest.mark.parametrize("N,V,K", [(40, 1000, 1000), (300, 64, 64), (9, 1, 1), (40, 1000, 999), (40, 5000, 100)])
def test_high_temperatures(N, V, K, T, dtype):
    h, w, z, index, g = _case(N, 64, V, K, dtype, 2.0)
    t = 2.0 * torch.randn(N, K, generator=g, device=DEV)
    rows, bound, dz = _expected(h, w, z, index, t, T)
    leaf = h.clone().requires_grad_()
    loss = E.linear_distillation(leaf, w, index, t, temperature=T, reduction="none")
    assert bool(((loss.double() - rows).abs() <= bound).all()), float(((loss.double() - rows).abs() / bound).max())
    if dtype is torch.float32:
        got, = torch.autograd.grad(loss.sum(), leaf)
        # T 2^-20 of q and of p, through V products and their sum
        q = torch.softmax(z / T, 1)
        size = (q + (dz / T - q).abs()) @ w.double().abs()
        assert bool(((got.double() - dz @ w.double()).abs() <= T * 2.0**-20 * size + 2.0**-20 * size).all())


@pytest.mark.parametrize("T", [0.5, 2.0, 100.0])
def test_a_student_that_is_the_teacher(T):
    """The loss of a teacher's own logits is a square of roundings, not a rounding."""
    h, w, z, index, _ = _case(50, 64, 700, 700, torch.float32, 2.0)
    t = z.gather(1, index).float()
    rows, bound, _ = _expected(h, w, z, index, t, T)
    got = E.linear_distillation(h, w, index, t, temperature=T, reduction="none")
    assert bool((got >= 0).all()) and bool(((got.double() - rows).abs() <= bound).all())
    assert float(got.max()) <= T * T * 1e-9


def test_all_tokens_named_in_part_twice_or_by_none():
    """Rows of as many entries as tokens, of which some name one twice or none: what they leave out counts."""
    h, w, z, index, g = _case(60, 64, 100, 100, torch.float32, 2.0)
    t = 2.0 * torch.randn(60, 100, generator=g, device=DEV)
    index[:20, 3] = index[:20, 70]
    index[20:40, 5] = -1
    T = 3.0
    teacher = torch.where(index >= 0, t.double() / T, -math.inf)
    logp = torch.log_softmax(teacher, 1)
    lq = torch.log_softmax(z / T, 1).gather(1, index.clamp(min=0))
    p = logp.exp()
    rows = T * T * torch.where(p > 0, p * (logp - lq), 0.0).sum(1)
    got = E.linear_distillation(h, w, index, t, temperature=T, reduction="none")
    # 64 products a logit, its size and a hundred terms: 400 roundings of numbers of size log V at most
    assert bool(((got.double() - rows).abs() <= T * T * 400 * U * math.log(100)).all())


@pytest.mark.parametrize("T", [1.0, 100.0, 1e4])
def test_of_logits_agrees(T):
    """The torch operations for heads that are more than a linear map, which sum in float64."""
    h, w, z, index, g = _case(40, 64, 500, 500, torch.float32, 2.0)
    t = 2.0 * torch.randn(40, 500, generator=g, device=DEV)
    rows, _, _ = _expected(h, w, z, index, t, T)
    got = logits_distillation(z.float(), index, t, T, "none")
    assert got.dtype is torch.float32
    # z in float32: u |z| of it, times the gradient, T (q - p), whose parts are |x| u T q; float64's own cancelling
    off = (z.abs() * U).amax(1) * (torch.softmax(z / T, 1).scatter_add(1, index, -torch.softmax(t.double() / T, 1)) * T
                                   ).abs().sum(1)
    assert bool(((got.double() - rows).abs() <= 2 * off + 2 * U * rows + T * T * 2.0**-44).all())
