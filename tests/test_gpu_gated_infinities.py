"""Gradients of ``gated_linear`` where an infinity stands in the last row of an operand: zeros behind it, which fill up
the last stage of a product, must not meet it (zero times an infinity is NaN)."""

import pytest
import torch

import ews_mi355x as E
from test_gpu_gated_linear import DTYPES, HALF_UNIT, U, _inputs

pytestmark = pytest.mark.gpu

INF = float("inf")


def _formula(x, w, b, gw, gb, up):
    x, w, b, gw, gb, up = (t.double() for t in (x, w, b, gw, gb, up))
    v, g = x @ w.t() + b, x @ gw.t() + gb
    s, r = torch.sigmoid(g), torch.sigmoid(-g)
    dv, dg = up * s, up * (v * (s * r))
    return dv @ w + dg @ gw, dv.t() @ x, dg.t() @ x


def _same(got, want, off):
    """Infinite and NaN where the formula is; else within ``off`` of the largest."""
    assert torch.equal(got.isnan(), want.isnan())
    there = want.isinf()
    assert torch.equal(got[there].double(), want[there])
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine)
    if bool(fine.any()):
        assert float((got[fine].double() - want[fine]).abs().max()) <= off * float(want[fine].abs().max())


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", [(7, 200, 40), (30, 192, 40), (60, 200, 41), (90, 200, 40), (90, 192, 40),
                                   (300, 520, 700), (300, 512, 700), (1030, 832, 4616)])
def test_the_last_row(N, H, F, dtype, joint):
    print(f"{N} {H} {F} {dtype} {joint}", flush=True)
    _check(N, H, F, dtype, joint, ((1, (F - 1, 9)), (3, (F - 1, 9)), (0, (N - 1, 5))))


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", [(90, 31, 40), (300, 16, 64), (70, 64, 4), (200, 64, 64), (2111, 32, 32)])
def test_narrow(N, H, F, dtype, joint):
    """Widths with kernels of their own; bfloat16's dv and dg have two planes there, the second none of an infinity."""
    print(f"{N} {H} {F} {dtype} {joint}", flush=True)
    _check(N, H, F, dtype, joint, ((1, (F - 1, 9)), (3, (1, 2)), (0, (N - 1, 5)), (0, (3, H - 1))))


def _check(N, H, F, dtype, joint, places):
    x, w, b, gw, gb, up = _inputs(N, H, F, dtype, joint=False)
    for tensor, at in places:
        ops = [t.clone() for t in (x, w, b, gw, gb)]
        ops[tensor][at] = INF
        want = _formula(*ops, up)
        if joint:
            leaves = [ops[0], torch.cat([ops[1], ops[3]]), torch.cat([ops[2], ops[4]])]
            leaves = [t.requires_grad_() for t in leaves]
            gx, gW, _ = torch.autograd.grad(E.gated_linear(*leaves), leaves, up)
            gv, gg = gW.chunk(2)
        else:
            leaves = [t.requires_grad_() for t in ops]
            gx, gv, _, gg, _ = torch.autograd.grad(E.gated_linear(*leaves), leaves, up)
        # a float32 sum's terms and, for bfloat16, dv's and dg's rounding and the result's, at random over a row
        for got, ref in zip((gx, gv, gg), want):
            _same(got, ref, 4 * HALF_UNIT[dtype] + (N + 2 * F + H) * U)
