"""Embedding lookup (csrc/ews_embed.hip) against its formula: the forward is one rounded product per number, so it is
compared bit for bit; a gradient row of c float32 sums is within (c + 1) 2^-24 of the sum of magnitudes, and half a unit
of its own type."""

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _inputs(shape, V, H, dtype, seed=0, kind="uniform"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = 1
    for s in shape:
        n *= s
    w = torch.randn(V, H, generator=g, device=DEV).to(dtype)
    if kind == "uniform":
        t = torch.randint(0, V, (n,), generator=g, device=DEV)
    elif kind == "same":
        t = torch.full((n,), V - 1, device=DEV)
    else:  # a few tokens are most of the text
        u = torch.rand(n, generator=g, device=DEV)
        t = (u**4 * V).long().clamp_(max=V - 1)
    return t.reshape(shape), w


def _forward_reference(t, w, scale):
    return (w.float()[t] * torch.tensor(scale, dtype=torch.float32, device=DEV)).to(w.dtype)


def _check_gradient(got, t, gout, V, scale, padding=None):
    t = t.reshape(-1)
    g = gout.reshape(t.numel(), -1).double()
    keep = (t >= 0) & (t < V)
    if padding is not None:
        keep &= t != padding
    H = g.shape[1]
    exact = torch.zeros(V, H, device=DEV, dtype=torch.float64).index_add_(0, t[keep], g[keep]) * scale
    total = torch.zeros(V, H, device=DEV, dtype=torch.float64).index_add_(0, t[keep], g[keep].abs()) * abs(scale)
    count = torch.zeros(V, device=DEV, dtype=torch.float64).index_add_(
        0, t[keep], torch.ones_like(t[keep], dtype=torch.float64))
    bound = (count + 2)[:, None] * 2.0**-24 * total + HALF_UNIT[got.dtype] * exact.abs() + 1e-37
    assert got.shape == exact.shape
    err = (got.double() - exact).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert not bool(got[count == 0].any())


CASES = [
    # tokens, V, H, which tokens
    ((1,), 1, 1, "uniform"),
    ((1,), 100003, 64, "uniform"),
    ((2, 3), 5, 3, "uniform"),
    ((31,), 2, 8, "uniform"),
    ((32,), 8, 130, "uniform"),
    ((33,), 300, 64, "same"),
    ((4, 64), 8, 32, "uniform"),
    ((4096,), 257, 24, "few"),
    ((4097,), 1025, 72, "few"),
    ((3, 3001), 5000, 520, "few"),
    ((9000,), 3, 16, "same"),
    ((20001,), 1, 5, "same"),
    ((5,), 40, 4100, "uniform"),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,V,H,kind", CASES)
def test_lookup_and_gradient(shape, V, H, kind, dtype):
    t, w = _inputs(shape, V, H, dtype, seed=len(shape) + V, kind=kind)
    for scale, padding, tok in ((1.0, None, t), (H**0.5, 0, t.int())):
        w.requires_grad_()
        out = E.embedding_lookup(tok, w, scale=scale, padding_idx=padding)
        assert out.dtype == dtype and out.shape == (*shape, H)
        assert torch.equal(out.detach(), _forward_reference(t, w.detach(), scale))
        gout = torch.randn(out.shape, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV).to(dtype)
        (grad,) = torch.autograd.grad(out, w, gout)
        assert grad.dtype == dtype
        _check_gradient(grad, t, gout, V, scale, padding)
        again = torch.autograd.grad(E.embedding_lookup(tok, w, scale=scale, padding_idx=padding), w, gout)[0]
        assert torch.equal(grad, again)  # no sum depends on the order of execution
        with torch.no_grad():
            assert torch.equal(E.embedding_lookup(tok, w, scale=scale), out.detach())


def test_all_tokens_are_padding():
    t = torch.zeros(100, dtype=torch.int64, device=DEV)
    w = torch.randn(7, 12, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(E.embedding_lookup(t, w, padding_idx=-7), w, torch.ones(100, 12, device=DEV))
    assert not bool(g.any())


def test_unknown_tokens_read_nothing():
    t = torch.tensor([3, -1, 9, 2**40, 0, -(2**33)], device=DEV)
    w = torch.randn(9, 20, device=DEV, requires_grad=True)
    out = E.embedding_lookup(t, w)
    assert torch.equal(out[[0, 4]], w[[3, 0]])
    assert bool(torch.isnan(out[[1, 2, 3, 5]]).all())
    gout = torch.ones_like(out)
    gout[[1, 2, 3, 5]] = float("nan")
    (g,) = torch.autograd.grad(out, w, gout)
    assert bool(torch.isfinite(g).all()) and float(g.sum()) == 40.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    big = torch.randn(50, 96, device=DEV).to(dtype)
    t = torch.randint(0, 50, (40, 2), device=DEV)
    for w in (big[:, :64], big[:, 1:33], big[::2, 3:30], big.t()[:50, :40], big[:, :1].expand(50, 16)):
        V = w.shape[0]
        tok = t.clamp(max=V - 1)
        for ids in (tok, tok[:, 0], tok.t()):
            assert torch.equal(E.embedding_lookup(ids, w), w[ids])
    # the gradient of a strided table, of an expanded cotangent and of a transposed one
    w = big[:, 1:33].detach().requires_grad_()
    out = E.embedding_lookup(t[:, 0], w, scale=0.5)
    for gout in (torch.ones((), device=DEV, dtype=dtype).expand(40, 32), torch.randn(32, 40, device=DEV).to(dtype).t()):
        (g,) = torch.autograd.grad(out, w, gout, retain_graph=True)
        _check_gradient(g, t[:, 0], gout, 50, 0.5)


def test_no_tokens_and_other_streams():
    w = torch.randn(6, 16, device=DEV, requires_grad=True)
    none = torch.empty(0, 4, dtype=torch.int64, device=DEV)
    out = E.embedding_lookup(none, w)
    assert out.shape == (0, 4, 16)
    assert not bool(torch.autograd.grad(out.sum(), w)[0].any())
    t = torch.randint(0, 6, (1000,), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = E.embedding_lookup(t, w)
        (g,) = torch.autograd.grad(out, w, torch.ones_like(out))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out.detach(), w.detach()[t])
    assert torch.equal(g[:, 0], torch.bincount(t, minlength=6).float())


def test_second_derivatives_are_refused():
    w = torch.randn(6, 16, device=DEV, requires_grad=True)
    out = E.embedding_lookup(torch.arange(6, device=DEV), w)
    gout = torch.ones_like(out, requires_grad=True)
    (g,) = torch.autograd.grad(out, w, gout, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), gout)


def test_refusals_on_the_device():
    w = torch.randn(6, 16, device=DEV)
    t = torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError, match="int64 or int32"):
        E.embedding_lookup(t.float(), w)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        E.embedding_lookup(t, w.double())
    with pytest.raises(ValueError, match="tokens are on"):
        E.embedding_lookup(t.cpu(), w)
    with pytest.raises(ValueError, match="outside a vocabulary"):
        E.embedding_lookup(t, w, padding_idx=6)
    with pytest.raises(ValueError, match="weight must be"):
        E.embedding_lookup(t, w[0])
