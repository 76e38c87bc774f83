"""What ``gated_linear`` keeps, what ``gated_scan`` leaves for its backward, and the scratch of both, between walls that
have to stay as they are."""

import pytest
import torch

import ews_mi355x as E
from ews_mi355x import gated, recurrence

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]
WALL = 1 << 16


@pytest.fixture
def walls(monkeypatch):
    made = []

    def walled(x, size):
        if not size:
            return None
        whole = torch.full((size + 2 * WALL,), 173, dtype=torch.uint8, device=DEV)
        made.append((whole, size))
        return whole[WALL:WALL + size]

    monkeypatch.setattr(gated, "_scratch", walled)
    monkeypatch.setattr(recurrence, "_scratch", walled)
    yield made
    torch.cuda.synchronize()
    assert made
    for whole, size in made:
        assert bool((whole[:WALL] == 173).all()) and bool((whole[WALL + size:] == 173).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", [(1, 5, 3), (1, 70, 65), (3, 65, 7), (31, 72, 130), (33, 72, 130), (64, 128, 100),
                                   (65, 128, 100), (300, 64, 200), (700, 128, 64), (90, 31, 40), (1030, 776, 4610),
                                   (4100, 1032, 6600)])
def test_linear(walls, N, H, F, dtype):
    print(f"{N} {H} {F} {dtype}", flush=True)
    for joint in (True, False):
        x, w = torch.randn(N, H, device=DEV).to(dtype), torch.randn(2 * F if joint else F, H, device=DEV).to(dtype)
        b = torch.randn(len(w), device=DEV).to(dtype)
        leaves = [t.requires_grad_() for t in (x, w, b, *([] if joint else [torch.randn_like(w)]))]
        y = E.gated_linear(*leaves, activation="silu")
        torch.autograd.grad(y, leaves, torch.randn_like(y))
        with torch.no_grad():
            E.gated_linear(*leaves, activation="silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["convex", "linear"])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (3, 2, 5), (2, 17, 70), (3, 200, 9), (2, 127, 33), (600, 17, 450),
                                   (1100, 18, 500), (128, 40, 516), (12, 260, 516), (24, 260, 516), (1, 2100, 3),
                                   (2, 4099, 40)])
def test_scan(walls, B, L, D, form, dtype):
    print(f"{B} {L} {D} {form} {dtype}", flush=True)
    x, gate = (torch.randn(B, L, D, device=DEV).to(dtype).requires_grad_() for _ in range(2))
    state = torch.randn(B, D, device=DEV, requires_grad=True)
    mask = torch.rand(B, L, device=DEV) < 0.7
    for m in (None, mask):
        h, last = E.gated_scan(x, gate, state=state, mask=m, form=form)
        torch.autograd.grad((h, last), (x, gate, state), (torch.randn_like(h), torch.randn_like(last)))
