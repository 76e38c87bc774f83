"""How often bfloat16 gradients of ``gated_linear`` are rounded, by their errors' lengths.

Rounding numbers of all mantissas m to bfloat16 leaves an error of 2^-8 / sqrt(3) sqrt(E[1 / m^2]) of their length, E[1
/ m^2] being 1/2 of uniform mantissas and 0.54 of logarithmic ones: r <= 1.75e-3 with 0.6. dv | dg are rounded once and
a product of them once more, at random: sqrt(2) r. (Sums kept in 16 bits would add 1 or 2 of v's and g's own, sqrt(3) r
at least.) Narrow maps have them in two planes: r. What is kept in 24 bits adds 2^-17, float32 sums (H + F) 2^-24.

The biases' gradients are sums of dv and dg before that, rounded once. They are F numbers, some 64, whose errors' length
the few largest decide, by where in their unit they lie: so each is held to half a unit of itself, 2^-8, and to 2^-15 of
the size of what is added (v's, g's and the activation's 2^-16, the float32 sum of N terms another (N + 8) 2^-24)."""

import math

import pytest
import torch

import ews_mi355x as E
from test_gpu_gated_linear import _inputs

pytestmark = pytest.mark.gpu

R = 2.0**-8 / math.sqrt(3) * math.sqrt(0.6)


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("N,H,F,roundings", [(300, 512, 700, 2), (30, 520, 1200, 2), (1030, 776, 4610, 2),
                                             (5000, 60, 64, 1)])
def test_roundings(N, H, F, roundings, act):
    print(f"{N} {H} {F} {act}", flush=True)
    x, w, b, gw, gb, up = _inputs(N, H, F, torch.bfloat16, joint=False)
    xd, V, b_, G, c_, d = (t.double() for t in (x, w, b, gw, gb, up))
    v, g = xd @ V.t() + b_, xd @ G.t() + c_
    s = torch.sigmoid(g)
    dv, dg = (d * s, d * v * s * (1 - s)) if act == "sigmoid" else (d * g * s, d * v * (s + g * s * (1 - s)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, gw, gb)]
    got = torch.autograd.grad(E.gated_linear(*leaves, activation=act), leaves, up)
    want = dv @ V + dg @ G, dv.t() @ xd, dv.sum(0), dg.t() @ xd, dg.sum(0)
    for name, a, r in zip("xVbGc", got, want):
        if name in "bc":
            size = (dv if name == "b" else dg).abs().sum(0)
            off = (a.double() - r).abs() / (2.0**-8 * r.abs() + (2.0**-15 + (N + 8) * 2.0**-24) * size)
            assert float(off.max()) <= 1, (name, float(off.max()))
            continue
        off = float((a.double() - r).norm() / r.norm())
        assert off <= math.sqrt(roundings) * R + 2.0**-15, (name, off)
