"""``gated_linear`` (csrc/ews_gated.hip) against its formula in float64 on the same (float32 or bfloat16) inputs.

Bounds, number by number. With u = 2^-24 a float32 sum of H products s_k is off by at most (H + 8) u sum |s_k| (the planes'
left-out products are 2 u of them), so v and g by ev and eg. An activation's own arithmetic: the logistic function's
argument z (g, or GELU's polynomial) is rounded four times at most, so the function by 4 u |z| of itself, its exponential,
sum, reciprocal and products by 12 u more; act and act' carry that of the numbers that they are formed of, and eg times the
next derivative (at most 1/4, 1.1, 1.13, 1 for act; 0.1, 0.5, 1.2 for act', and where relu's kink is nearer than eg
anything up to |v|). What is kept for the backward, and each dv and dg, is rounded to the type once (bfloat16: half a unit,
2^-8, each). A gradient is off by the sum of these times the other operand, its float32 sum, and half a unit."""

import math

import pytest
import torch

import ews_mi355x as E
from gated_shapes import SHARED, TILES

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
HALF_UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
ACTS = ["sigmoid", "silu", "gelu", "relu"]
DTYPES = [torch.float32, torch.bfloat16]


def _inputs(N, H, F, dtype, joint=True, bias=True, seed=0, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + N + 31 * H + 7 * F)

    def randn(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device=DEV)).to(dtype)

    x, up = randn(N, H), randn(N, F)
    rows = 2 * F if joint else F
    w, b = randn(rows, H, scale=spread / math.sqrt(H)), randn(rows, scale=0.5) if bias else None
    if joint:
        return x, w, b, None, None, up
    return x, w, b, randn(F, H, scale=spread / math.sqrt(H)), randn(F, scale=0.5) if bias else None, up


def _act(g, name):
    """act, act', and how far their own arithmetic may be off."""
    if name == "relu":
        on = (g > 0).double()
        return g * on, on, 0 * g, 0 * g
    u, du = g, torch.ones_like(g)
    if name == "gelu":
        u = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)
        du = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    p, q = torch.sigmoid(u), torch.sigmoid(-u)
    off = (4 * u.abs() + 12) * U
    if name == "sigmoid":
        return p, p * q, off * p, 2 * off * p * q
    return g * p, p + g * p * q * du, off * (g * p).abs(), 2 * off * (p + (g * p * q * du).abs())


_BEND = {"sigmoid": (0.25, 0.1), "silu": (1.1, 0.5), "gelu": (1.13, 1.2), "relu": (1.0, 0.0)}


def _reference(x, w, b, gw, gb, up, name):
    """{name: (value, bound)} of y and the gradients of x, V, b, G, c."""
    half = HALF_UNIT[x.dtype]
    H = x.shape[1]
    xd, wd = x.double(), w.double()
    F = wd.shape[0] if gw is not None else wd.shape[0] // 2
    V, G = (wd, gw.double()) if gw is not None else (wd[:F], wd[F:])
    zero = torch.zeros(F, device=DEV, dtype=torch.float64)
    bv = zero if b is None else b.double()[:F]
    bg = (zero if gb is None else gb.double()) if gw is not None else (zero if b is None else b.double()[F:])
    v, g = xd @ V.t() + bv, xd @ G.t() + bg
    ev = (H + 8) * U * (xd.abs() @ V.abs().t() + bv.abs())
    eg = (H + 8) * U * (xd.abs() @ G.abs().t() + bg.abs())
    act, slope, ra, rs = _act(g, name)
    la, ls = _BEND[name]
    ea, es = la * eg + ra, ls * eg + rs
    if name == "relu":
        es = torch.where(g.abs() <= eg, torch.ones_like(g), es)
    y = v * act
    out = {"y": (y, act.abs() * ev + v.abs() * ea + ev * ea + (half + U) * y.abs())}
    d = up.double()
    q = v * slope
    ep, eq = ea + half * act.abs(), slope.abs() * ev + v.abs() * es + ev * es + (half + U) * q.abs()
    dv, dg = d * act, d * q
    edv, edg = d.abs() * ep * (1 + half) + half * dv.abs(), d.abs() * eq * (1 + half) + half * dg.abs()
    dx = dv @ V + dg @ G
    mass = dv.abs() @ V.abs() + dg.abs() @ G.abs()
    out["x"] = dx, edv @ V.abs() + edg @ G.abs() + (2 * F + 8) * U * mass + half * dx.abs()
    N = x.shape[0]
    for key, dz, e in (("V", dv, edv), ("G", dg, edg)):
        dw, db = dz.t() @ xd, dz.sum(0)
        out[key] = dw, e.t() @ xd.abs() + (N + 8) * U * (dz.abs().t() @ xd.abs()) + half * dw.abs()
        out["b" + key] = db, e.sum(0) + (N + 8) * U * dz.abs().sum(0) + half * db.abs()
    return out


def _close(got, want, what):
    value, bound = want
    assert got.shape == value.shape, what
    err = (got.double() - value).abs()
    ok = err <= bound + 1e-36
    assert bool(ok.all()), (what, float((err / (bound + 1e-36)).max()), int((~ok).sum()))


def _check(x, w, b, gw, gb, up, name):
    want = _reference(x, w, b, gw, gb, up, name)
    with torch.no_grad():
        y = E.gated_linear(x, w, b, gw, gb, activation=name)
    assert y.dtype is x.dtype
    _close(y, want["y"], "y alone")
    leaves = {k: t.detach().clone().requires_grad_() for k, t in (("x", x), ("w", w), ("b", b), ("gw", gw), ("gb", gb))
              if t is not None}
    y = E.gated_linear(*(leaves.get(k) for k in ("x", "w", "b", "gw", "gb")), activation=name)
    _close(y.detach(), want["y"], "y")
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), up)))
    _close(grads["x"], want["x"], "grad x")
    if gw is None:
        _close(grads["w"], tuple(torch.cat(t) for t in zip(want["V"], want["G"])), "grad weight")
        if b is not None:
            _close(grads["b"], tuple(torch.cat(t) for t in zip(want["bV"], want["bG"])), "grad bias")
    else:
        for key, n in (("w", "V"), ("b", "bV"), ("gw", "G"), ("gb", "bG")):
            if key in grads:
                _close(grads[key], want[n], f"grad {n}")
    return y.detach(), grads


SHAPES = [
    (1, 1, 1), (1, 64, 64), (3, 5, 7), (2, 72, 130), (17, 64, 100), (33, 40, 24), (64, 128, 8), (65, 64, 65), (130, 200, 16),
    (257, 72, 515), (700, 24, 33), (2111, 32, 32), (63, 1032, 40), (1000, 33, 31), (999, 31, 64), (70, 64, 4), (5000, 60, 64),
    (140000, 8, 12), (3, 65, 7), (130, 70, 2), (1, 65, 65), (129, 128, 200),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", SHAPES)
def test_values_and_gradients(N, H, F, dtype):
    print(f"{N} {H} {F} {dtype}", flush=True)
    for i, name in enumerate(ACTS):
        _check(*_inputs(N, H, F, dtype, joint=i % 2 == 0, bias=i < 2, spread=2.0), name)


@pytest.mark.parametrize("joint", [True, False])
@pytest.mark.parametrize("name,N,H,F", list(TILES))
def test_every_tile(name, N, H, F, joint):
    print(f"{name} {N} {H} {F} {joint}", flush=True)
    _check(*_inputs(N, H, F, getattr(torch, name), joint=joint), "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", list(SHARED))
def test_shared_tiles(N, H, F, dtype):
    print(f"{N} {H} {F} {dtype}", flush=True)
    _check(*_inputs(N, H, F, dtype), "gelu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 33, 48, 64])
@pytest.mark.parametrize("H,F", [(8, 16), (31, 50), (512, 100), (1030, 37), (1096, 130)])
def test_few_rows(N, H, F, dtype):
    """Rows that are read straight into the matrix instructions: widths of whole and cut eights, outputs of cut sixteens."""
    for joint in (True, False):
        x, w, b, gw, gb, up = _inputs(N, H, F, dtype, joint=joint)
        with torch.no_grad():
            y = E.gated_linear(x, w, b, gw, gb, activation="gelu")
        _close(y, _reference(x, w, b, gw, gb, up, "gelu")["y"], f"joint={joint}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [5, 200])
def test_layouts(dtype, N):
    """Rows apart, off their 16-byte addresses, turned; weights of different strides; three axes; one bias alone."""
    x, w, b, gw, gb, up = _inputs(N, 128, 96, dtype, joint=False)
    base = _check(x, w, b, gw, gb, up, "sigmoid")

    def apart(t, cols):
        wide = torch.full((t.shape[0], cols), 7.0, device=DEV, dtype=dtype)
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    def off(t):
        flat = torch.empty(t.numel() + 1, device=DEV, dtype=dtype)[1:].view(t.shape)
        return flat.copy_(t)

    want = _reference(x, w, b, gw, gb, up, "sigmoid")
    for x2, w2, g2 in ((apart(x, 136), apart(w, 144), apart(gw, 144)), (x, apart(w, 144), gw), (x, apart(w, 131), gw),
                       (off(x), w, gw), (x, off(w), gw), (x, w, off(gw)), (apart(x, 129), off(w), off(gw)),
                       (x.t().contiguous().t(), w.t().contiguous().t(), gw)):
        got = _check(x2, w2, b, g2, gb, up, "sigmoid")
        _close(got[0], want["y"], "y")
    if N % 5 == 0:
        y = E.gated_linear(x.view(5, N // 5, 128), w, b, gw, gb)
        assert y.shape == (5, N // 5, 96) and torch.equal(y.view(N, 96), E.gated_linear(x, w, b, gw, gb))
    _check(x, w, b, gw, None, up, "relu")
    _check(x, w, None, gw, gb, up, "relu")
    assert base


@pytest.mark.parametrize("dtype", DTYPES)
def test_some_gradients(dtype):
    x, w, b, gw, gb, up = _inputs(70, 64, 40, dtype, joint=False)
    want = _reference(x, w, b, gw, gb, up, "silu")
    keys = dict(x="x", w="V", b="bV", gw="G", gb="bG")
    given = dict(x=x, w=w, b=b, gw=gw, gb=gb)
    for some in (["x"], ["w"], ["gw"], ["b"], ["gb"], ["x", "gw"], ["w", "b"]):
        leaves = {k: (t.clone().requires_grad_() if k in some else t) for k, t in given.items()}
        y = E.gated_linear(*leaves.values(), activation="silu")
        for k, g in zip(some, torch.autograd.grad(y, [leaves[k] for k in some], up)):
            _close(g, want[keys[k]], k)


@pytest.mark.parametrize("name", ACTS)
def test_far_gates(name):
    """Gates of any finite size, and infinite or NaN x in rows of their own."""
    x, w, b, gw, gb, up = _inputs(80, 64, 32, torch.float32, joint=False)
    for scale in (30.0, 1e4, 1e12):
        g2 = gw * scale
        want = _reference(x, w, b, g2, gb, up, name)
        leaves = [t.clone().requires_grad_() for t in (x, w, b, g2, gb)]
        y = E.gated_linear(*leaves, activation=name)
        _close(y.detach(), want["y"], f"y {scale}")
        for key, g in zip(("x", "V", "bV", "G", "bG"), torch.autograd.grad(y, leaves, up)):
            assert bool(g.isfinite().all())
            _close(g, want[key], f"{key} {scale}")
    bad = x.clone()
    bad[3, 5], bad[70] = float("nan"), float("nan")
    for rows in (slice(0, 80), slice(0, 64)):
        with torch.no_grad():
            y = E.gated_linear(bad[rows], w, b, gw, gb, activation=name)
            fine = E.gated_linear(x[rows], w, b, gw, gb, activation=name)
        hit = torch.zeros(80, dtype=torch.bool, device=DEV)
        hit[[3, 70]] = True
        assert bool(y[hit[rows]].isnan().all()) and torch.equal(y[~hit[rows]], fine[~hit[rows]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,F", [(7, 200, 40), (60, 200, 40), (90, 200, 40), (7, 31, 40), (90, 31, 40)])
def test_infinities(N, H, F, dtype):
    """Infinite x, and weights, where the formula gives infinities, not NaN: rows straight into registers, tiles, narrow."""
    x, w, b, gw, gb, up = _inputs(N, H, F, dtype, joint=False)
    inf = float("inf")
    for tensor, at, value in ((x, (3, 5), inf), (x, (N - 1, H - 1), -inf), (w, (4, H - 1), inf), (w, (F - 1, 0), -inf)):
        bad, badw = x.clone(), w.clone()
        (bad if tensor is x else badw)[at] = value
        v, g = bad.double() @ badw.double().t() + b.double(), bad.double() @ gw.double().t() + gb.double()
        want = v * torch.sigmoid(g)
        with torch.no_grad():
            y = E.gated_linear(bad, badw, b, gw, gb)
            fine = E.gated_linear(x, w, b, gw, gb)
        hit = ~v.isfinite() | ~g.isfinite()
        assert bool(hit.any()) and torch.equal(y[~hit], fine[~hit])
        assert torch.equal(y[hit].isnan(), want[hit].isnan())
        there = hit & ~want.isnan()
        assert torch.equal(y[there].double(), want[there])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [7, 30, 60, 90])
def test_gradients_of_infinite_weights(N, dtype):
    """An infinite weight makes x's gradient infinite or NaN where the formula's is."""
    x, w, b, gw, gb, up = _inputs(N, 200, 40, dtype, joint=False)
    w[4, 9] = float("inf")
    xd, V, G = x.double(), w.double(), gw.double()
    v, s = xd @ V.t() + b.double(), torch.sigmoid(xd @ G.t() + gb.double())
    want = (up.double() * s) @ V + (up.double() * v * s * (1 - s)) @ G
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(E.gated_linear(leaf, w, b, gw, gb), leaf, up)
    assert not bool(want.isfinite().any()) and torch.equal(got.isnan(), want.isnan())
    there = ~want.isnan()
    assert torch.equal(got[there].double(), want[there])


def test_gradient_against_differences():
    for name in ("sigmoid", "silu", "gelu"):
        x, w, b, _, _, up = _inputs(90, 32, 24, torch.float32)
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = E.gated_linear(*leaves, activation=name)
        grads = torch.autograd.grad(y, leaves, up)
        step = 2.0**-7
        for k, g in enumerate(grads):
            way = torch.randn(g.shape, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV)
            way /= way.norm()
            values = []
            for sign in (1, -1):
                t = [x, w, b]
                t[k] = t[k] + sign * step * way
                with torch.no_grad():
                    values.append((E.gated_linear(*t, activation=name).double() * up.double()).sum())
            got, want = float((values[0] - values[1]) / (2 * step)), float((g.double() * way.double()).sum())
            # 2160 results of some 40 roundings each, at random, over 2^-6; and step^2 / 6 of a third derivative that a
            # direction of length one, |x| about 6 a row, takes to 6^3 in a row at most
            assert abs(got - want) <= 2160**0.5 * 40 * U * 4 / 2.0**-6 + step**2 / 6 * 216 * 10


def test_the_same_bits_twice_and_on_another_stream():
    x, w, b, gw, gb, up = _inputs(700, 136, 300, torch.bfloat16, joint=False)
    want = _check(x, w, b, gw, gb, up, "gelu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, gw, gb)]
        y = E.gated_linear(*leaves, activation="gelu")
        once = torch.autograd.grad(y, leaves, up, retain_graph=True)
        twice = torch.autograd.grad(y, leaves, up)
    side.synchronize()
    assert torch.equal(y.detach(), want[0])
    for a, r, t in zip(once, want[1].values(), twice):
        assert torch.equal(a, r) and torch.equal(a, t)


def test_scratch_holds_what_a_call_writes(monkeypatch):
    """Scratch and what is kept between walls that have to stay as they are."""
    from ews_mi355x import gated as module

    walls = []

    def walled(x, size):
        whole = torch.full((size + 8192,), 173, dtype=torch.uint8, device=DEV)
        walls.append((whole, size))
        return whole[4096:4096 + size]

    monkeypatch.setattr(module, "_scratch", walled)
    for N, H, F, dtype in ((1, 5, 3, torch.float32), (33, 72, 130, torch.bfloat16), (300, 64, 200, torch.float32),
                           (700, 128, 64, torch.bfloat16), (2111, 32, 32, torch.float32)):
        _check(*_inputs(N, H, F, dtype), "silu")
        _check(*_inputs(N, H, F, dtype, joint=False), "relu")
    torch.cuda.synchronize()
    for whole, size in walls:
        assert bool((whole[:4096] == 173).all()) and bool((whole[4096 + size:] == 173).all())


def test_empty():
    w = torch.randn(12, 5, device=DEV, requires_grad=True)
    x = torch.zeros(0, 5, device=DEV, requires_grad=True)
    y = E.gated_linear(x, w)
    assert y.shape == (0, 6)
    gx, gw = torch.autograd.grad(y.sum(), [x, w])
    assert gx.shape == x.shape and not gw.any()
    assert E.gated_linear(torch.zeros(2, 0, 5, device=DEV), w.detach()).shape == (2, 0, 6)


def test_second_derivatives_are_refused():
    x, w, b, _, _, up = _inputs(9, 16, 8, torch.float32)
    x.requires_grad_()
    g, = torch.autograd.grad(E.gated_linear(x, w, b), x, up, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_device():
    x, w, b, gw, gb, _ = _inputs(8, 16, 6, torch.float32, joint=False)
    with pytest.raises(TypeError, match="weight is"):
        E.gated_linear(x, w.bfloat16(), b, gw, gb)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        E.gated_linear(x.half(), w.half())
    with pytest.raises(ValueError, match="bias is on"):
        E.gated_linear(x, w, b.cpu(), gw, gb)
