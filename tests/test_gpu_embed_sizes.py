"""Embedding lookup's gradient at the sizes where its parts change: vocabularies of which a sorting workgroup owns many
tokens or that need more than 256 of those workgroups, and tables of more rows and column tiles than a grid's x holds.

A gradient row of c float32 sums is within (c + 1) 2^-24 of the sum of magnitudes, and half a unit of its own type."""

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _check(grad, tokens, gout, scale):
    """The rows of grad that have tokens, in float64; all others are zero."""
    rows, back = tokens.unique(return_inverse=True)
    g = gout.double() * scale
    exact = torch.zeros(len(rows), g.shape[1], device=DEV, dtype=torch.float64).index_add_(0, back, g)
    total = torch.zeros_like(exact).index_add_(0, back, g.abs())
    count = torch.bincount(back).double()[:, None]
    bound = (count + 2) * 2.0**-24 * total + HALF_UNIT[grad.dtype] * exact.abs() + 1e-37
    assert bool(((grad[rows].double() - exact).abs() <= bound).all())
    rest = 0
    for part in grad.split(1 << 22):  # a huge table's counts, a few rows at a time
        rest += int(part.count_nonzero())
    assert rest == int(grad[rows].count_nonzero())


@pytest.mark.parametrize("n", [200, 1000])
def test_more_rows_than_a_grid_holds(n):
    """2^25 rows of 65 bfloat16 numbers (two column tiles each): 2^26 units, which x alone does not hold."""
    V, H = 1 << 25, 65
    g = torch.Generator(device=DEV).manual_seed(n)
    t = torch.randint(0, V, (n,), generator=g, device=DEV)
    t[:7] = torch.tensor([0, V - 1, V - 1, V // 2, (1 << 24) - 1, 1 << 24, V - 2], device=DEV)
    w = torch.zeros(V, H, device=DEV, dtype=torch.bfloat16)
    w[t] = torch.randn(n, H, generator=g, device=DEV).bfloat16()
    w.requires_grad_()
    out = E.embedding_lookup(t, w, scale=0.5)
    assert torch.equal(out.detach(), (w.detach()[t].float() * 0.5).bfloat16())
    gout = torch.randn(n, H, generator=g, device=DEV).bfloat16()
    (grad,) = torch.autograd.grad(out, w, gout)
    _check(grad, t, gout, 0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,H,half", [(9000, 60000, 24, False), (30001, 131072, 16, True), (5000, 131073, 40, False),
                                        (40003, 200003, 20, True), (3000, 1000003, 8, True)])
def test_vocabularies_of_many_sorting_workgroups(n, V, H, half, dtype):
    """A workgroup that owns 256 and 512 tokens; 512 to 2048 workgroups. half: half the text is one token, more than a
    wavefront lists."""
    g = torch.Generator(device=DEV).manual_seed(V)
    t = torch.randint(0, V, (n,), generator=g, device=DEV)
    t[:6] = torch.tensor([0, V - 1, V // 2, 511, 512, 255], device=DEV)
    if half:
        t[torch.rand(n, generator=g, device=DEV) < 0.5] = V - 3
    w = torch.randn(V, H, generator=g, device=DEV).to(dtype).requires_grad_()
    gout = torch.randn(n, H, generator=g, device=DEV).to(dtype)
    for tokens in (t, t.int()):
        out = E.embedding_lookup(tokens, w, scale=2.5)
        (grad,) = torch.autograd.grad(out, w, gout)
        _check(grad, t, gout, 2.5)
    (again,) = torch.autograd.grad(E.embedding_lookup(t, w, scale=2.5), w, gout)
    assert torch.equal(grad, again)
