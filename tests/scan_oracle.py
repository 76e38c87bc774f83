"""The gated recurrence step by step in float64, its gradients by hand, and how far float32 arithmetic may be off."""

import torch

HALF32 = 2.0**-24  # half a step of float32, relative


def recurrence(x, gate, state, mask, form, dh, dlast):
    """Values and bounds {name: (value, bound)} of h, last, dx, dgate, dstate; everything float64 on the CPU.

    The bounds carry every rounding through the recurrence itself. One step's factor a has the relative error
    (|g| + 6) half steps: exp(-g) takes g log2(e), whose rounding is |g| half steps of the result, an exponential and a
    reciprocal of two each, and a sum; a state adds two roundings more. Steps are composed in tiles before they are
    applied: a state's path goes through a thread's steps, the wavefront's composition (six levels) and the
    workgroup's, and each composition rounds a product and a sum again: four times the bound of the steps alone."""
    B, L, D = x.shape
    convex = form == "convex"
    a = torch.sigmoid(gate) if convex else gate.clone()
    take = torch.sigmoid(-gate) if convex else torch.ones_like(gate)
    loose = (4 * HALF32) * ((gate.abs() if convex else torch.zeros_like(gate)) + 8)
    x = x.clone()
    if mask is not None:
        off = ~mask
        a[off], take[off], x[off], loose[off] = 1.0, 0.0, 0.0, 4 * HALF32
    h = torch.zeros(B, D, dtype=torch.float64) if state is None else state
    e = torch.zeros_like(h)
    hs, es, befores = [], [], []
    for t in range(L):
        befores.append((h, e))
        e = a[:, t].abs() * e + loose[:, t] * (a[:, t].abs() * h.abs() + (take[:, t] * x[:, t]).abs())
        h = a[:, t] * h + take[:, t] * x[:, t]
        hs.append(h)
        es.append(e)
    lam = torch.zeros_like(h)
    m = torch.zeros_like(h) if dlast is None else dlast
    em = torch.zeros_like(h)
    dx, dg, ex, eg = [], [], [], []
    for t in range(L - 1, -1, -1):
        u = dh[:, t]
        lam = u + m
        el = em + HALF32 * 4 * (u.abs() + m.abs())
        before, eb = befores[t]
        gx = lam * take[:, t]
        dx.append(gx)
        ex.append(el * take[:, t] + loose[:, t] * gx.abs())
        slope = (before - x[:, t]) * a[:, t] * take[:, t] if convex else before * (take[:, t] if mask is not None else 1)
        slack = a[:, t].abs() * take[:, t] * (eb + HALF32 * (before.abs() + x[:, t].abs())) if convex else eb
        dg.append(lam * slope)
        eg.append(el * slope.abs() + lam.abs() * slack + 3 * loose[:, t] * (lam * slope).abs())
        m = a[:, t] * lam
        em = a[:, t].abs() * el + loose[:, t] * m.abs()
    out = {"h": (torch.stack(hs, 1), torch.stack(es, 1)), "last": (h, e), "dx": (torch.stack(dx[::-1], 1), torch.stack(ex[::-1], 1)),
           "dgate": (torch.stack(dg[::-1], 1), torch.stack(eg[::-1], 1)), "dstate": (m, em)}
    return out


def assert_near(got, want, bound, name=""):
    """Within the bound and the rounding to got's type."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.detach().double().cpu()
    allowed = bound + half * (want.abs() + bound) + 1e-37
    worst = ((got - want).abs() / allowed).max() if got.numel() else torch.zeros(())
    assert got.shape == want.shape, name
    assert float(worst) <= 1.0, f"{name}: {float(worst):.3g} of what rounding explains"
