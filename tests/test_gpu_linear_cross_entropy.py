"""Linear cross entropy (csrc/ews_loss.hip) against its formula in float64 on the same (float32 or bfloat16) inputs.

Bounds, number by number. With unit u = 2^-24 and S = sum_k |h_k w_k|, a logit is off by at most dz = (H + 8) u S
(float32 sums, the planes' left-out products at most 2 u S), so a loss by 2 max dz + 8 u (1 + |z|), and a
probability by the factor 1 + e, e = 2 max dz + 16 u + 2 u max |z|. dz carries e of its p, and where it is held in
bfloat16 the rounding of the probability and its own, 2^-9 each. A gradient is then off by the sum of these times the
other operand's magnitude, its float32 sum's (K + 8) u of the summed magnitudes, and half a unit of its own type."""

import math

import pytest
import torch
import torch.nn.functional as F

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
HALF_UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _inputs(N, H, V, dtype, bias=None, ignored=0.0, seed=0, spread=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed + N + 31 * H + 7 * V)
    w = (torch.randn(V, H, generator=g, device=DEV) * (spread / math.sqrt(H))).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device=DEV)
    h = (torch.randn(N, H, generator=g, device=DEV) + 3.0 * torch.rand(N, 1, generator=g, device=DEV) * w[t]).to(dtype)
    b = None if bias is None else (0.5 * torch.randn(V, generator=g, device=DEV)).to(bias)
    t[torch.rand(N, generator=g, device=DEV) < ignored] = -100
    return h, w, b, t


def _reference(h, w, b, t, reduction, upstream=None, grads=True, planes=1):
    """(loss, gh, gw, gb), their bounds; kept rows only are looked at."""
    V = w.shape[0]
    keep = t != -100
    x, wd = h.double()[keep], w.double()
    tk = t[keep]
    z = x @ wd.t()
    if b is not None:
        z = z + b.double()
    n = tk.numel()
    H = w.shape[1]
    zerr = (H + 8) * U * (x.abs() @ wd.abs().t()).max(1).values if n else torch.zeros(0, device=DEV).double()
    lse = torch.logsumexp(z, 1)
    rows = lse - z[torch.arange(n, device=DEV), tk]
    zmag = torch.where(torch.isfinite(z), z, torch.zeros_like(z)).abs().max(1).values if n else zerr
    rerr = 2 * zerr + 8 * U * (1 + zmag)
    g = torch.ones(n, device=DEV, dtype=torch.float64)
    if reduction == "mean":
        g /= max(1, n)
    if upstream is not None:
        g = g * (upstream.double()[keep] if reduction == "none" else float(upstream))
    if reduction == "none":
        loss = torch.zeros(t.numel(), device=DEV, dtype=torch.float64)
        loss[keep] = rows
        lerr = torch.zeros_like(loss)
        lerr[keep] = rerr
    else:
        scale = 1.0 / max(1, n) if reduction == "mean" else 1.0
        loss = rows.sum() * scale
        lerr = rerr.sum() * scale + U * loss.abs()
    if not grads:
        return loss, lerr
    p = torch.softmax(z, 1)
    d = p.clone()
    d[torch.arange(n, device=DEV), tk] -= 1.0
    d *= g[:, None]
    e = 2 * zerr + 16 * U + 2 * U * zmag
    derr = p * (e * g.abs())[:, None] + 4 * U * d.abs()
    if h.dtype == torch.bfloat16 and planes == 1:
        derr = derr + 2 * 2.0**-8 * 1.01 * d.abs()
    elif h.dtype == torch.bfloat16:  # probabilities as 16-bit logarithms, then 16 bits of dz
        derr = derr + 1.1 * 2.0**-10.5 * p * g.abs()[:, None] + 2.0**-16 * d.abs()
    gh = torch.zeros_like(h, dtype=torch.float64)
    gh[keep] = d @ wd
    herr = torch.zeros_like(gh)
    herr[keep] = derr @ wd.abs() + (V + 8) * U * (d.abs() @ wd.abs())
    gw = d.t() @ x
    werr = derr.t() @ x.abs() + (n + 8) * U * (d.abs().t() @ x.abs())
    out, bound = [loss, gh, gw], [lerr, herr + HALF_UNIT[h.dtype] * gh.abs(), werr + HALF_UNIT[w.dtype] * gw.abs()]
    if b is not None:
        gb = d.sum(0)
        out.append(gb)
        bound.append(derr.sum(0) + (n + 8) * U * d.abs().sum(0) + HALF_UNIT[b.dtype] * gb.abs())
    return out, bound


def _close(got, want, bound, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    ok = err <= bound + 1e-36
    assert bool(ok.all()), (what, float((err / (bound + 1e-36)).max()), int((~ok).sum()))


def _check(h, w, b, t, reduction="mean", upstream=None):
    wrt = [x.detach().clone().requires_grad_() for x in (h, w, b) if x is not None]
    bb = wrt[2] if b is not None else None
    loss = E.linear_cross_entropy(wrt[0], wrt[1], t, bias=bb, reduction=reduction)
    assert loss.dtype == torch.float32
    up = upstream
    if up is None and reduction == "none":
        up = torch.rand(t.shape, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) + 0.5
    got = torch.autograd.grad(loss, wrt, up)
    want, bound = _reference(h, w, b, t, reduction, up)
    for name, a, r, e in zip(("loss", "grad_hidden", "grad_weight", "grad_bias"), (loss.detach(), *got), want, bound):
        _close(a, r, e, name)
    with torch.no_grad():
        score = E.linear_cross_entropy(h, w, t, bias=b, reduction=reduction)
    _close(score, want[0], bound[0], "score")
    return loss.detach(), got


SHAPES = [
    (1, 1, 1), (1, 64, 8), (3, 5, 7), (2, 64, 4099), (32, 72, 300), (33, 64, 129), (64, 64, 256), (65, 100, 300),
    (130, 128, 1000), (257, 72, 515), (300, 200, 2049), (1030, 64, 13000), (5, 520, 70000), (2111, 24, 8),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V", SHAPES)
def test_loss_and_gradients(N, H, V, dtype):
    print(f"loss N={N} H={H} V={V} {dtype}", flush=True)
    _check(*_inputs(N, H, V, dtype))
    _check(*_inputs(N, H, V, dtype, bias=dtype, ignored=0.3), reduction="sum")
    _check(*_inputs(N, H, V, dtype, bias=torch.float32, ignored=0.3), reduction="none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_results(dtype):
    """Enough results for the largest tiles in both gradients."""
    print(f"wide {dtype}", flush=True)
    _check(*_inputs(10050, 1032, 300, dtype, ignored=0.1))
    _check(*_inputs(300, 1030, 13001, dtype, bias=dtype))


@pytest.mark.parametrize("dtype,N", [(torch.float32, 3000), (torch.bfloat16, 11000)])
def test_rows_in_chunks(dtype, N):
    """More rows than are kept at a time, also where the later chunks hold ignored rows alone."""
    print(f"chunks {dtype} N={N}", flush=True)
    h, w, b, t = _inputs(N, 40, 100003, dtype, bias=dtype, ignored=0.05)
    _check(h, w, b, t)
    t[N // 4:] = -100
    _check(h, w, b, t)


@pytest.mark.parametrize("N,H,V,reduction", [(1, 72, 67, "none"), (8, 128, 67, "none"), (33, 64, 500, "none"),
                                             (200, 136, 1003, "none"), (256, 64, 300, "none"), (2, 128, 67, "mean"),
                                             (16, 200, 1000, "sum")])
def test_few_rows_of_bfloat16_are_rounded_once(N, H, V, reduction):
    """Where few rows add up, dz has sixteen bits: the gradients are off by little more than their own rounding."""
    h, w, b, t = _inputs(N, H, V, torch.bfloat16, bias=torch.float32, ignored=0.1 if N > 4 else 0.0)
    wrt = [x.requires_grad_() for x in (h, w, b)]
    loss = E.linear_cross_entropy(h, w, t, bias=b, reduction=reduction)
    up = torch.rand(N, device=DEV) + 0.5 if reduction == "none" else None
    got = torch.autograd.grad(loss, wrt, up)
    want, bound = _reference(*(x.detach() for x in wrt), t, reduction, up, planes=2)
    for a, r, e, name in zip(got, want[1:], bound[1:], ("hidden", "weight", "bias")):
        _close(a, r, e, f"grad_{name}")


def test_scores_in_chunks():
    """Rows of a call without gradients beyond those whose slabs are kept at a time; a row's loss is its own, so some
    rows are looked at. A row's sum goes through up to 200 additions one after another."""
    h, w, b, t = _inputs(22000, 16, 100003, torch.bfloat16, bias=torch.float32, ignored=0.05)
    with torch.no_grad():
        got = E.linear_cross_entropy(h, w, t, bias=b, reduction="none")
    for lo in (0, 10980, 11240, 21230, 21950):
        rows = slice(lo, lo + 50)
        want, bound = _reference(h[rows], w, b, t[rows], "none", None, grads=False)
        _close(got[rows], want, bound + 200 * U, f"rows from {lo}")


@pytest.mark.parametrize("N,V", [(250, 1 << 22), (500, 1 << 20)])
def test_few_rows_of_a_huge_vocabulary(N, V):
    """The probabilities' planes of 250 rows and 2^22 tokens are wider than 32-bit offsets reach; 500 rows of 2^20 are
    done in chunks with W read as it is. A row's sum goes through up to 600 additions one after another."""
    h, w, b, t = _inputs(N, 8, V, torch.float32)
    h.requires_grad_()
    loss = E.linear_cross_entropy(h, w, t, reduction="none")
    (got,) = torch.autograd.grad(loss, h, torch.ones_like(loss))
    for lo in (0, N // 2 + 10, N - 4):
        rows = slice(lo, lo + 4)
        want, bound = _reference(h[rows].detach(), w, b, t[rows], "none", torch.ones(4, device=DEV))
        _close(loss[rows].detach(), want[0], bound[0] + 600 * U, f"loss from {lo}")
        _close(got[rows], want[1], bound[1], f"grad_hidden from {lo}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_ignored_rows_are_not_read(dtype, reduction):
    h, w, b, t = _inputs(100, 96, 200, dtype, bias=dtype)
    t[::3] = -100
    clean = _check(h, w, b, t, reduction)
    bad = h.clone()
    bad[0], bad[3], bad[6] = float("nan"), float("inf"), torch.finfo(dtype).min
    wrt = [x.clone().requires_grad_() for x in (bad, w, b)]
    loss = E.linear_cross_entropy(*wrt[:2], t, bias=wrt[2], reduction=reduction)
    up = torch.rand(t.shape, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) + 0.5
    got = torch.autograd.grad(loss, wrt, up if reduction == "none" else None)
    assert torch.equal(loss, clean[0])
    for a, r in zip(got, clean[1]):
        assert torch.equal(a, r)
    assert not bool(got[0][::3].any())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_every_row_ignored(reduction):
    h, w, b, t = _inputs(70, 64, 150, torch.float32, bias=torch.float32)
    t[:] = -100
    h[:] = float("nan")
    wrt = [x.requires_grad_() for x in (h, w, b)]
    loss = E.linear_cross_entropy(h, w, t, bias=b, reduction=reduction)
    got = torch.autograd.grad(loss, wrt, torch.ones_like(loss))
    assert not bool(loss.any()) and not any(bool(x.any()) for x in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_taken_out_by_the_bias(dtype):
    h, w, b, t = _inputs(90, 64, 500, dtype, bias=torch.float32)
    t[(t >= 200) & (t < 330)] = 7  # leaves whole slabs of the vocabulary without a token
    out = torch.ones(500, dtype=torch.bool, device=DEV)
    out[t] = False
    b[out] = -float("inf")
    loss, got = _check(h, w, b, t)
    assert not bool(got[1][out].any()) and not bool(got[2][out].any())
    # the type's lowest value in every entry: the logits keep their order, nothing overflows
    low = torch.full((500,), torch.finfo(torch.float32).min, device=DEV)
    with torch.no_grad():
        value = E.linear_cross_entropy(h, w, t, bias=low)
    assert abs(float(value) - math.log(500.0)) < 1e-4  # float32 holds no difference beside it: a uniform row
    # a row whose every token is taken out, and one whose own is
    b2 = torch.full((500,), -float("inf"), device=DEV)
    assert bool(torch.isnan(E.linear_cross_entropy(h, w, t, bias=b2, reduction="none")).all())
    b2[:] = 0.0
    b2[t[0]] = -float("inf")
    rows = E.linear_cross_entropy(h, w, t, bias=b2, reduction="none")
    assert float(rows[0]) == float("inf") and bool(torch.isfinite(rows[t != t[0]]).all())


def test_unknown_targets_give_nan():
    h, w, b, t = _inputs(10, 64, 50, torch.float32)
    t[3], t[4] = 50, -7
    rows = E.linear_cross_entropy(h, w, t, reduction="none")
    assert bool(torch.isnan(rows[[3, 4]]).all()) and int(torch.isnan(rows).sum()) == 2
    assert bool(torch.isnan(E.linear_cross_entropy(h, w, t)))
    assert bool(torch.isfinite(E.linear_cross_entropy(h, w, torch.where(t == 50, t, t.clamp(min=0)), ignore_index=50)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_confident_and_large_logits(dtype):
    """Targets of probability near one (their gradient is the small rest) and logits of hundreds."""
    for spread in (8.0, 60.0):
        h, w, b, t = _inputs(150, 64, 400, dtype, spread=spread)
        _check(h, w, b, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    h, w, b, t = _inputs(60, 72, 210, dtype, bias=dtype)
    big = torch.zeros(300, 200, device=DEV, dtype=dtype)
    big[:60, 3:75] = h
    wide = torch.zeros(210, 136, device=DEV, dtype=dtype)
    wide[:, 64:136] = w
    want = E.linear_cross_entropy(h, w, t, bias=b, reduction="none")
    for hh, ww in ((big[:60, 3:75], wide[:, 64:136]), (h.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(E.linear_cross_entropy(hh, ww, t, bias=b, reduction="none"), want)
    got = E.linear_cross_entropy(h.view(4, 15, 72), w, t.view(4, 15).int(), bias=b, reduction="none")
    assert got.shape == (4, 15) and torch.equal(got.reshape(-1), want)
    # one row for all: its gradient is the sum over the rows
    one = h[:1].detach().requires_grad_()
    loss = E.linear_cross_entropy(one.expand(60, 72), w, t, bias=b, reduction="sum")
    (g,) = torch.autograd.grad(loss, one)
    (want_all, bound) = _reference(h[:1].expand(60, 72), w, b, t, "sum")
    slack = bound[1].sum(0, keepdim=True) + 60 * HALF_UNIT[dtype] * want_all[1].abs().sum(0, keepdim=True)
    _close(g, want_all[1].sum(0, keepdim=True), slack, "expanded hidden")


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_some_gradients_and_upstream(reduction):
    h, w, b, t = _inputs(77, 64, 333, torch.float32, bias=torch.float32, ignored=0.2)
    up = torch.tensor(-2.5, device=DEV) if reduction == "mean" else torch.randn(77, device=DEV)
    want, bound = _reference(h, w, b, t, reduction, up)
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, True, False)):
        xs = [x.clone().requires_grad_(n) for x, n in zip((h, w, b), need)]
        loss = E.linear_cross_entropy(xs[0], xs[1], t, bias=xs[2], reduction=reduction)
        wrt = [x for x in xs if x.requires_grad]
        first = torch.autograd.grad(loss, wrt, up, retain_graph=True)
        second = torch.autograd.grad(loss, wrt, up)
        for got, again, (r, e) in zip(first, second, [(r, e) for r, e, n in zip(want[1:], bound[1:], need) if n]):
            _close(got, r, e + 2 * U * r.abs(), "gradient")
            assert torch.equal(got, again)


def test_gradient_against_differences():
    """Central differences of the float64 formula's loss along random directions, and of this loss itself."""
    h, w, b, t = _inputs(40, 64, 90, torch.float32, bias=torch.float32, ignored=0.1)
    xs = [x.clone().requires_grad_() for x in (h, w, b)]
    grads = torch.autograd.grad(E.linear_cross_entropy(xs[0], xs[1], t, bias=xs[2]), xs)
    g = torch.Generator(device=DEV).manual_seed(3)
    for k in range(3):
        d = [torch.randn(x.shape, generator=g, device=DEV) if i == k else torch.zeros_like(x)
             for i, x in enumerate((h, w, b))]
        slope = sum(float((a.double() * x.double()).sum()) for a, x in zip(grads, d))
        s = 1e-4
        up, down = ([x.double() + s * y.double() for x, y in zip((h, w, b), d)],
                    [x.double() - s * y.double() for x, y in zip((h, w, b), d)])
        f = [float(F.cross_entropy(x @ y.t() + z, t)) for x, y, z in (up, down)]
        assert abs((f[0] - f[1]) / (2 * s) - slope) < 1e-5 * max(1.0, abs(slope))
        s = 1e-2  # the loss in float32: its rounding over 2 s, and the third derivative's s^2
        f = [float(E.linear_cross_entropy(h + q * s * d[0], w + q * s * d[1], t, bias=b + q * s * d[2]))
             for q in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * s) - slope) < 5e-3 * max(1.0, abs(slope))


def test_another_stream_and_the_same_bits():
    h, w, b, t = _inputs(500, 128, 3001, torch.bfloat16, bias=torch.float32, ignored=0.1)
    first = _check(h, w, b, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _check(h, w, b, t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], second[0])
    for a, r in zip(first[1], second[1]):
        assert torch.equal(a, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 70, 301])
def test_kept_probabilities_and_new_ones_give_the_same_bits(N, dtype):
    """The first backward of the rows' own losses forms the gradients from what the forward kept, a second one (whose
    upstream may differ) computes it again."""
    h, w, b, t = _inputs(N, 136, 500, dtype, bias=torch.float32, ignored=0.2 if N > 1 else 0.0)
    wrt = [x.requires_grad_() for x in (h, w, b)]
    up = torch.rand(N, device=DEV) + 0.5
    rows = E.linear_cross_entropy(h, w, t, bias=b, reduction="none")
    first = torch.autograd.grad(rows, wrt, up, retain_graph=True)
    other = torch.autograd.grad(rows, wrt, up * 2.0, retain_graph=True)
    again = torch.autograd.grad(rows, wrt, up)
    for a, c, d in zip(first, other, again):
        assert torch.equal(a, d) and torch.equal(c, a * 2.0)
    rows = E.linear_cross_entropy(h, w, t, bias=b, reduction="none")
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(rows, wrt, up)


SCRATCH = [(141, 396, 1980), (256, 64, 1000), (200, 1000, 333), (33, 257, 4001), (7, 4096, 700), (300, 130, 900)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V", SCRATCH)
def test_scratch_holds_what_a_call_writes(N, H, V, dtype, monkeypatch):
    """Beyond the bytes that the library asks for, a workspace stays as it was, whatever the address of the weight makes
    of the plan."""
    from ews_mi355x import loss as module

    spaces = []

    def workspace(self, train):
        size = module.nat.load().ews_loss_workspace_bytes(self.desc, train)
        whole = torch.full((size + (64 << 20),), 91, dtype=torch.uint8, device=DEV)
        spaces.append((whole, size))
        return whole[:size]

    monkeypatch.setattr(module._Call, "workspace", workspace)
    h, w, b, t = _inputs(N, H, V, dtype, bias=torch.float32, ignored=0.3)
    odd = torch.empty(V * H + 1, device=DEV, dtype=dtype)[1:].view(V, H)
    for weight in (w, odd.copy_(w)):
        weight = weight.detach().requires_grad_()
        for reduction in ("none", "mean"):
            hidden = h.detach().requires_grad_()
            rows = E.linear_cross_entropy(hidden, weight, t, bias=b, reduction=reduction)
            torch.autograd.grad(rows, [hidden, weight], torch.ones_like(rows))
        with torch.no_grad():
            E.linear_cross_entropy(h, weight, t, bias=b)
    torch.cuda.synchronize()
    assert len(spaces) == 6
    for whole, size in spaces:
        assert bool((whole[size:] == 91).all())


def test_second_derivatives_are_refused():
    h, w, b, t = _inputs(6, 16, 20, torch.float32, bias=torch.float32)
    h.requires_grad_()
    (g,) = torch.autograd.grad(E.linear_cross_entropy(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), h)


def test_no_rows():
    w = torch.randn(9, 16, device=DEV, requires_grad=True)
    h = torch.empty(0, 16, device=DEV, requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device=DEV)
    for reduction in ("mean", "sum", "none"):
        loss = E.linear_cross_entropy(h, w, t, reduction=reduction)
        gh, gw = torch.autograd.grad(loss.sum(), [h, w])
        assert gh.shape == (0, 16) and not bool(gw.any()) and float(loss.detach().sum()) == 0.0


def test_refusals_on_the_device():
    h, w, b, t = _inputs(6, 16, 20, torch.float32, bias=torch.float32)
    for bad, kind in ((dict(hidden=h.bfloat16()), TypeError), (dict(hidden=h.double()), TypeError),
                      (dict(weight=w.half()), TypeError), (dict(targets=t.float()), TypeError),
                      (dict(bias=b.double()), TypeError), (dict(targets=t[:5]), ValueError),
                      (dict(bias=b[:5]), ValueError), (dict(hidden=h[:, :8]), ValueError),
                      (dict(weight=w[0]), ValueError), (dict(targets=t.cpu()), ValueError),
                      (dict(reduction="max"), ValueError), (dict(hidden=h.cpu()), RuntimeError)):
        with pytest.raises(kind):
            E.linear_cross_entropy(**{**dict(hidden=h, weight=w, targets=t, bias=b), **bad})
