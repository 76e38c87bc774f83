"""``gated_scan`` of the convex form with infinite inputs, states and upstream gradients: a gate that is not shut keeps
an infinity, however many steps' product of gates has left float32's range; one of the other sign makes NaN."""

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

INF = float("inf")
SIZES = [(3, 2, 5), (2, 127, 33), (3, 200, 9), (2, 257, 16), (128, 40, 516), (12, 260, 516), (24, 260, 516),
         (1, 2100, 3), (2, 4099, 40), (600, 17, 450)]


def _steps(x, gate, state, dh):
    """States, and the gradients of x, gate and state, one step after the other in float64."""
    a, take = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    h, hs, before = state.double(), [], []
    for t in range(x.shape[1]):
        before.append(h)
        h = a[:, t] * h + take[:, t] * x[:, t].double()
        hs.append(h)
    m, dx, dg = torch.zeros_like(h), [], []
    for t in range(x.shape[1] - 1, -1, -1):
        l = dh[:, t].double() + m
        dx.append(l * take[:, t])
        dg.append(l * take[:, t] * (a[:, t] * (before[t] - x[:, t].double())))
        m = a[:, t] * l
    return torch.stack(hs, 1), torch.stack(dx[::-1], 1), torch.stack(dg[::-1], 1), m


def _alike(got, want, what):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got.isinf(), want.isinf()), what
    there = want.isinf()
    assert torch.equal(got[there], want[there]), what
    # finite ones: no more than a hint that they are the right numbers, which other tests hold to their roundings
    fine = want.isfinite()
    assert bool(((got[fine] - want[fine]).abs() <= 0.02 * (1 + want[fine].abs())).all()), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D", SIZES)
def test_infinities_stay(B, L, D, dtype):
    print(f"{B} {L} {D} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(B + L + D)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    for where in ("x", "state", "dh", "both signs"):
        x, gate = randn(B, L, D).to(dtype), (randn(B, L, D) - 3).to(dtype)
        state, dh = randn(B, D), randn(B, L, D).to(dtype)
        if where == "x":
            x[0, 0, 0], x[-1, L // 3, D - 1] = INF, -INF
        elif where == "state":
            state[0, 0], state[-1, D - 1] = INF, -INF
        elif where == "dh":
            dh[0, L - 1, 0], dh[-1, L // 2, D - 1] = INF, -INF
        else:
            x[0, 0, 0], x[0, L - 1, 0] = INF, -INF
        want = _steps(x, gate, state, dh)
        leaves = [t.clone().requires_grad_() for t in (x, gate, state)]
        h, last = E.gated_scan(*leaves)
        _alike(h.detach(), want[0], f"h {where}")
        _alike(last.detach(), want[0][:, -1], f"last {where}")
        for name, a, r in zip(("dx", "dgate", "dstate"), torch.autograd.grad(h, leaves, dh), want[1:]):
            _alike(a, r, f"{name} {where}")
