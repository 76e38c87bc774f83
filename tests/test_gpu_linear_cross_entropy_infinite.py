"""Infinities in the head's weight or the hidden rows (csrc/ews_loss.hip): a logit is the sum of its products, so an
infinite factor gives an infinity of the products' sign, or NaN beside a zero or an infinity of the other sign. A logit
of -inf takes its token out of the row's softmax; one of +inf, or NaN, makes the row's loss NaN.

The oracle is the formula in float64 on the CPU. Where its value is finite the bounds are those of finite inputs, with S
the sum of the finite products' magnitudes: a logit (H + 8) 2^-24 S (plus bfloat16's half unit where a gradient is
rounded to it), a loss twice that and 8 * 2^-24 (1 + |z|)."""

import math

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
INF = float("inf")


def _inputs(N, H, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + N + 31 * H + 7 * V)
    w = (torch.randn(V, H, generator=g) * (1.5 / math.sqrt(H))).to(dtype)
    h = torch.randn(N, H, generator=g).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    return h, w, t


def _oracle(h, w, t):
    """Rows' losses and their bounds, and the logits."""
    x, y = h.double(), w.double()
    z = x @ y.t()
    finite = [torch.where(torch.isfinite(a), a, torch.zeros_like(a)).abs() for a in (x, y)]
    S = (finite[0] @ finite[1].t()).max(1).values
    zmag = torch.where(torch.isfinite(z), z, torch.zeros_like(z)).abs().max(1).values
    rows = torch.arange(len(t))
    top = z.max(1, keepdim=True).values
    # a row of +inf or NaN, or of nothing but -inf, has no probabilities
    loss = torch.where(torch.isfinite(top[:, 0]), torch.log(torch.exp(z - top).sum(1)) + top[:, 0] - z[rows, t],
                       torch.full_like(top[:, 0], float("nan")))
    return loss, 2 * (w.shape[1] + 8) * U * S + 8 * U * (1 + zmag), z


def _same(got, want, bound, what):
    got = got.detach().double().cpu()
    for name, kind in (("NaN", torch.isnan), ("+inf", lambda a: a == INF), ("-inf", lambda a: a == -INF)):
        assert torch.equal(kind(got), kind(want)), f"{what}: {name} at other places"
    ok = torch.isfinite(want)
    bound = bound.expand_as(want)
    assert bool(((got - want).abs() <= bound)[ok].all()), what


def _run(h, w, t, reduction="none"):
    with torch.no_grad():
        return E.linear_cross_entropy(h.to(DEV), w.to(DEV), t.to(DEV), reduction=reduction)


# float32 W as it is (one, few and more rows; rows of W at multiples of 16 bytes or not; stages that H does not fill)
# and in planes (128 x 128 and 256 x 256 tiles); bfloat16 as it is and packed
SHAPES = [(1, 64, 300), (20, 72, 300), (20, 77, 301), (100, 96, 1000), (100, 61, 1001), (700, 64, 6500),
          (520, 333, 16500), (300, 77, 500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V", SHAPES)
def test_losses(N, H, V, dtype):
    print(f"infinite N={N} H={H} V={V} {dtype}", flush=True)
    h, w, t = _inputs(N, H, V, dtype)
    g = torch.Generator().manual_seed(1)
    # column 0 of h is positive, the last one negative: their products' signs are known
    h[:, 0], h[:, H - 1] = h[:, 0].abs() + 0.5, -h[:, H - 1].abs() - 0.5
    for k in range(0, V, max(1, V // 40)):  # tokens taken out
        w[k, 0 if k % 2 else H - 1] = -INF if k % 2 else INF
    w[V - 1, H - 1] = INF
    w[V - 1, 0] = -INF
    loss, bound, z = _oracle(h, w, t)
    assert bool((z[:, V - 1] == -INF).all()) and not bool(torch.isnan(z).any())
    _same(_run(h, w, t), loss, bound, "tokens taken out")
    # some rows see an infinity of a random sign, a zero beside it, an infinity on both sides, NaN
    w[3, 5], h[:, 7 % H] = INF, torch.randn(N, generator=g).to(dtype)
    w[5, 7 % H] = -INF
    h[N // 2, 5] = 0.0
    h[N // 3, 9] = INF
    w[7, 9] = INF
    h[N - 1, 2] = float("nan") if N > 1 else h[N - 1, 2]
    loss, bound, z = _oracle(h, w, t)
    _same(_run(h, w, t), loss, bound, "infinities of both signs")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V", SHAPES[1:])
def test_gradients(N, H, V, dtype):
    """Tokens taken out by an infinite weight: no probability, a zero row of the weight's gradient; hidden's gradient is
    0 times infinity in the columns of the infinities and finite in the others."""
    h, w, t = _inputs(N, H, V, dtype, seed=1)
    h[:, 0], h[:, H - 1] = h[:, 0].abs() + 0.5, -h[:, H - 1].abs() - 0.5
    out = torch.zeros(V, dtype=torch.bool)
    out[::11] = True
    out[V - 1] = True
    t = torch.where(out[t], torch.ones_like(t), t)
    w[out, 0] = -INF
    w[V - 1, H - 1] = INF
    loss, bound, z = _oracle(h, w, t)
    x, y = (a.to(DEV).requires_grad_() for a in (h, w))
    rows = E.linear_cross_entropy(x, y, t.to(DEV), reduction="none")
    _same(rows, loss, bound, "losses")
    up = torch.rand(N, generator=torch.Generator().manual_seed(2)) + 0.5
    gx, gw = torch.autograd.grad(rows, [x, y], up.to(DEV))
    d = torch.softmax(z, 1)
    d[torch.arange(N), t] -= 1.0
    d *= up.double()[:, None]
    e = (bound[:, None] + 16 * U) * 2
    half = U if dtype == torch.float32 else 2.0**-8
    derr = d.abs() * (e + (4 * U if dtype == torch.float32 else 2.0**-8 * 1.01))
    if dtype == torch.bfloat16:
        derr = derr + 1.1 * 2.0**-10.5 * (d.abs() + 2.0 * torch.nn.functional.one_hot(t, V))
    want = d.t() @ h.double()
    _same(gw, want, derr.t() @ h.double().abs() + (N + 8) * U * (d.abs().t() @ h.double().abs()) + half * want.abs(),
          "weight's gradient")
    assert not bool(gw[out.to(DEV)].any())
    bad = torch.isinf(w).any(0)
    assert bool(torch.isnan(gx[:, bad.to(DEV)]).all())
    y0 = torch.where(torch.isinf(w), torch.zeros_like(w), w).double()
    want = d @ y0
    bound = derr @ y0.abs() + (V + 8) * U * (d.abs() @ y0.abs()) + half * want.abs()
    ok = ~bad
    _same(gx[:, ok.to(DEV)], want[:, ok], bound[:, ok], "hidden's gradient")


def test_numbers_past_the_first_plane():
    """Float32 numbers that bfloat16 would round to infinity stay finite."""
    h, w, t = _inputs(40, 64, 500, torch.float32)
    h[:, 3] = 0.0
    w[:, 3] = torch.finfo(torch.float32).max
    w[7, 4], h[:, 4] = -3.4e38, 1e-37
    for N in (1, 40):
        loss, bound, _ = _oracle(h[:N], w, t[:N])
        _same(_run(h[:N], w, t[:N]), loss, bound, "as it is")
    big = h.repeat(15, 1)
    wide = torch.cat([w] * 14)
    loss, bound, _ = _oracle(big, wide, t.repeat(15))
    _same(_run(big, wide, t.repeat(15)), loss, bound, "planes")
