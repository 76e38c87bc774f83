"""The logistic function of float32 gates alone: x = 1 and V = 1 make y = act(g), for every kernel that forms it.

An exponential and a reciprocal of one unit (2 half units of 2^-24) each, its argument's second part (rounded twice, of
a part that is 2^-24 |g|: nothing), their sum and products, and y's own rounding: 8 half units, at any |g| up to 80."""

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24


@pytest.mark.parametrize("N", [1, 70, 200])
@pytest.mark.parametrize("H,F", [(1, 60), (1, 2000), (66, 2000)])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_far_gates_keep_their_digits(N, H, F, act):
    """Few rows, tiles and narrow maps; the other columns of x are zero."""
    g = torch.linspace(-80, 80, F, device=DEV)
    x, v, w = torch.zeros(N, H, device=DEV), torch.zeros(F, H, device=DEV), torch.zeros(F, H, device=DEV)
    x[:, 0], v[:, 0], w[:, 0] = 1.0, 1.0, g
    p, q = torch.sigmoid(g.double()), torch.sigmoid(-g.double())
    want, slope = (p, p * q) if act == "sigmoid" else (g.double() * p, p + g.double() * p * q)
    c = torch.zeros(F, device=DEV, requires_grad=True)
    y = E.gated_linear(x, v, None, w, c, activation=act)
    with torch.no_grad():
        alone = E.gated_linear(x, v, None, w, c, activation=act)
    for got in (y.detach(), alone):
        assert float(((got.double() - want).abs() / want.abs().clamp(min=1e-37)).max()) <= 8 * U + U
    if act == "sigmoid":  # silu's slope is a sum of both signs
        grad, = torch.autograd.grad(y, c, torch.ones_like(y))
        # a product of the two, and the sum of N equal numbers
        assert float(((grad.double() - N * slope).abs() / (N * slope)).max()) <= (2 * 8 + 1 + N) * U
