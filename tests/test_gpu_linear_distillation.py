"""Distillation from a teacher's largest logits (csrc/ews_loss.hip) against its formula in float64 on the same inputs.

Bounds as in the cross entropy's tests, whose kernels it shares: with u = 2^-24 and S = sum_k |h_k w_k| a logit is off by
at most dz = (H + 8) u S, over T, so log q by e = 2 dz / T + 16 u + 2 u max |z| / T and q by the factor 1 + e. The
teacher's exponents (t - max) / T are rounded twice (the difference and its product with a rounded factor: 3 u of them),
exp and the quotient take a few u, the float32 sum K u: a share p is off by ep = (3 |t - max| / T + K + 16) u of itself,
its logarithm by the same number. dz carries e of q and ep of p; in bfloat16 the rounding of the kept probability and its
own, 2^-9 of each entry's parts."""

import math

import pytest
import torch

import ews_mi355x as E
from loss_shapes import TILES

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
HALF_UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _inputs(N, H, V, K, dtype, bias=None, holes=0.2, seed=0, near=False, logits=torch.float32):
    """near: a row's entries are neighbours, so that they lie in one tile."""
    g = torch.Generator(device=DEV).manual_seed(seed + N + 31 * H + 7 * V + K)
    w = (torch.randn(V, H, generator=g, device=DEV) * (1.5 / math.sqrt(H))).to(dtype)
    order = torch.arange(V, device=DEV) if near else torch.randperm(V, generator=g, device=DEV)
    index = order[(torch.randint(0, V, (N, 1), generator=g, device=DEV) + torch.arange(K, device=DEV)) % V]
    h = (torch.randn(N, H, generator=g, device=DEV)
         + 3.0 * torch.rand(N, 1, generator=g, device=DEV) * w[index[:, 0]].float()).to(dtype)
    t = (3.0 * torch.randn(N, K, generator=g, device=DEV)).to(logits)
    index[torch.rand(N, K, generator=g, device=DEV) < holes] = -1
    if N > 3:
        index[::4] = -1  # rows without an entry
    b = None if bias is None else (0.5 * torch.randn(V, generator=g, device=DEV)).to(bias)
    return h, w, b, index, t


def _reference(h, w, b, index, t, T, reduction, upstream=None, planes=1):
    """The loss, the gradients and their bounds; rows with an entry only are looked at."""
    (V, H), (N, K) = w.shape, index.shape
    has = (index >= 0) & (t != -math.inf)
    keep = has.any(1)
    x, wd, idx, has = h.double()[keep], w.double(), index[keep], has[keep]
    n = x.shape[0]
    teacher = t.double()[keep].masked_fill(~has, -math.inf) / T
    z = x @ wd.t() if b is None else x @ wd.t() + b.double()
    z = z / T
    logq = torch.log_softmax(z, 1)
    logp = torch.log_softmax(teacher, 1)
    p = logp.exp()
    at = torch.where(has, idx, 0).clamp(max=V - 1)
    lq = logq.gather(1, at)
    lp = torch.where(p > 0, logp, 0.0)
    each = torch.where(p > 0, p * (lp - lq), 0.0)
    rows = T * T * each.sum(1)
    zerr = (H + 8) * U * (x.abs() @ wd.abs().t()).amax(1) / T
    zmag = torch.where(torch.isfinite(z), z, 0.0).abs().amax(1)
    e = 2 * zerr + 16 * U + 2 * U * zmag
    far = torch.where(has, teacher.amax(1, keepdim=True) - teacher, 0.0)
    ep = (3 * far + K + 16) * U
    size = torch.where(p > 0, p * (lp.abs() + lq.abs() + 1), 0.0)
    rerr = T * T * ((p * e[:, None]).sum(1) + (size * (ep + (K + 8) * U)).sum(1))
    g = torch.ones(n, device=DEV, dtype=torch.float64)
    if reduction == "mean":
        g /= max(1, n)
    if upstream is not None:
        g = g * (upstream.double()[keep] if reduction == "none" else float(upstream))
    if reduction == "none":
        loss, lerr = torch.zeros(N, device=DEV, dtype=torch.float64), torch.zeros(N, device=DEV, dtype=torch.float64)
        loss[keep], lerr[keep] = rows, rerr + U * rows.abs()
    else:
        scale = 1.0 / max(1, n) if reduction == "mean" else 1.0
        loss, lerr = rows.sum() * scale, (rerr.sum() + 2 * U * rows.abs().sum()) * scale
    share = torch.zeros_like(z).scatter_add_(1, at, p)
    slack = torch.zeros_like(z).scatter_add_(1, at, p * (ep + 4 * U))
    q = logq.exp()
    gt = (T * g)[:, None]
    d = gt * (q - share)
    derr = gt.abs() * (q * (e[:, None] + 4 * U) + slack) + 4 * U * d.abs()
    if h.dtype == torch.bfloat16 and planes == 1:
        derr = derr + 2 * 2.0**-8 * 1.01 * d.abs()
    elif h.dtype == torch.bfloat16:
        derr = derr + gt.abs() * 1.1 * 2.0**-10.5 * q + 2.0**-16 * d.abs()
    gh, herr = torch.zeros_like(h, dtype=torch.float64), torch.zeros_like(h, dtype=torch.float64)
    gh[keep] = d @ wd
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


def _check(h, w, b, index, t, T=1.0, reduction="mean", upstream=None, planes=1):
    wrt = [x.detach().clone().requires_grad_() for x in (h, w, b) if x is not None]
    loss = E.linear_distillation(wrt[0], wrt[1], index, t, bias=wrt[2] if b is not None else None, temperature=T,
                                 reduction=reduction)
    assert loss.dtype == torch.float32
    up = upstream
    if up is None and reduction == "none":
        up = torch.rand(index.shape[:-1], generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) + 0.5
    got = torch.autograd.grad(loss, wrt, up)
    want, bound = _reference(h, w, b, index, t, T, reduction, up, planes)
    for name, a, r, e in zip(("loss", "grad_hidden", "grad_weight", "grad_bias"), (loss.detach(), *got), want, bound):
        _close(a, r, e, name)
    with torch.no_grad():
        score = E.linear_distillation(h, w, index, t, bias=b, temperature=T, reduction=reduction)
    _close(score, want[0], bound[0], "score")
    return loss.detach(), got


SHAPES = [
    (1, 1, 1, 1), (1, 64, 8, 8), (3, 5, 7, 2), (2, 64, 4099, 64), (32, 72, 300, 65), (33, 64, 129, 129), (64, 64, 256, 3),
    (65, 100, 300, 100), (130, 128, 1000, 1), (257, 72, 515, 256), (300, 200, 2049, 1000), (1030, 64, 13000, 31),
    (5, 520, 70000, 1024), (2111, 24, 8, 5),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V,K", SHAPES)
def test_loss_and_gradients(N, H, V, K, dtype):
    print(f"{N} {H} {V} {K} {dtype}", flush=True)
    _check(*_inputs(N, H, V, K, dtype, bias=dtype), T=2.0)
    _check(*_inputs(N, H, V, K, dtype, near=True, holes=0.0), reduction="none", T=0.7)


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("name,N,H,V,reduction", list(TILES))
def test_every_tile(name, N, H, V, reduction, near):
    """The products' tiles are those of the cross entropy of the same sizes."""
    K = 20 if V > 100000 else 150
    print(f"{name} {N} {H} {V} {reduction} {near}", flush=True)
    _check(*_inputs(N, H, V, K, getattr(torch, name), near=near), reduction=reduction, T=1.5)


@pytest.mark.parametrize("dtype,N", [(torch.float32, 3000), (torch.bfloat16, 11000)])
def test_rows_in_chunks(dtype, N):
    print(f"chunks {dtype} N={N}", flush=True)
    h, w, b, index, t = _inputs(N, 40, 100003, 17, dtype, bias=dtype)
    _check(h, w, b, index, t, T=2.0)
    index[N // 4:] = -1
    _check(h, w, b, index, t, reduction="none")


@pytest.mark.parametrize("N,H,V,reduction", [(1, 72, 67, "none"), (33, 64, 500, "none"), (256, 64, 300, "none"),
                                             (2, 128, 67, "mean"), (16, 200, 1000, "sum")])
def test_few_rows_of_bfloat16_are_rounded_once(N, H, V, reduction):
    h, w, b, index, t = _inputs(N, H, V, 9, torch.bfloat16, bias=torch.float32)
    _check(h, w, b, index, t, reduction=reduction, planes=2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_one_entry_is_cross_entropy(reduction, dtype):
    h, w, b, index, t = _inputs(130, 72, 515, 1, dtype, bias=torch.float32, holes=0.1)
    outs = []
    for fn in (lambda *x: E.linear_distillation(x[0], x[1], index, t, bias=x[2], reduction=reduction),
               lambda *x: E.linear_cross_entropy(x[0], x[1], index[:, 0], bias=x[2], ignore_index=-1,
                                                 reduction=reduction)):
        leaves = [x.clone().requires_grad_() for x in (h, w, b)]
        loss = fn(*leaves)
        outs.append((loss.detach(), *torch.autograd.grad(loss, leaves)))
    for a, r in zip(*outs):
        assert torch.equal(a, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_token_named_twice(dtype):
    """Its entries count on their own, next to each other or not, also all of a row's the same."""
    h, w, b, index, t = _inputs(70, 72, 600, 12, dtype, bias=dtype, holes=0.1)
    index[:, 7] = index[:, 2]
    index[:, 8] = index[:, 2]
    index[5] = 3
    _check(h, w, b, index, t, T=2.0)
    _check(h, w, b, index, t, reduction="none")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_what_is_no_entry_is_not_used(reduction):
    h, w, b, index, t = _inputs(60, 64, 300, 6, torch.float32, bias=torch.float32, holes=0.4)
    want = _check(h, w, b, index, t, reduction=reduction)
    off = index < 0
    junk = t.clone()
    junk[off] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device=DEV).repeat(off.sum())[:off.sum()]
    far = index.clone()
    far[off] = -(1 << 40)
    gone = index.clone()  # the same entries taken out by their logits
    gone[off] = 7
    out = t.masked_fill(off, -float("inf"))
    h2 = h.clone()
    h2[off.all(1)] = float("nan")
    for args in ((h, w, b, far, junk), (h2, w, b, far, junk), (h, w, b, gone, out)):
        leaves = [x.clone().requires_grad_() for x in args[:3]]
        loss = E.linear_distillation(leaves[0], leaves[1], args[3], args[4], bias=leaves[2], reduction=reduction)
        up = None if reduction != "none" else torch.rand(
            60, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) + 0.5
        got = torch.autograd.grad(loss, leaves, up)
        for a, r in zip((loss.detach(), *got), (want[0], *want[1])):
            assert torch.equal(a, r)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_has_an_entry(reduction):
    h, w, b, index, t = _inputs(9, 64, 30, 3, torch.bfloat16, bias=torch.bfloat16)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    loss = E.linear_distillation(h, w, torch.full_like(index, -1), t, bias=b, reduction=reduction)
    assert not loss.any()
    for g in torch.autograd.grad(loss, leaves, torch.ones_like(loss)):
        assert not g.any()


def test_lowest_logits_and_far_ones():
    """Logits of the type's lowest value are entries; so much below the largest they have no probability. A row of
    nothing else is uniform over them."""
    h, w, b, index, t = _inputs(40, 64, 200, 8, torch.float32, holes=0.0)
    t[:, 3:] = torch.finfo(torch.float32).min
    t[1] = torch.finfo(torch.float32).min
    _check(h, w, b, index, t.clamp(min=-1e30), T=2.0)
    got = E.linear_distillation(h, w, index, t, reduction="none")
    want = E.linear_distillation(h, w, index, t.clamp(min=-1e30), reduction="none")
    assert torch.equal(got, want)


def test_unknown_tokens_give_nan():
    h, w, b, index, t = _inputs(30, 64, 100, 4, torch.float32)
    index[7, 2] = 100
    index[13, 0] = 1 << 40
    with torch.no_grad():
        loss = E.linear_distillation(h, w, index, t, reduction="none")
    bad = torch.zeros(30, dtype=torch.bool, device=DEV)
    bad[[7, 13]] = True
    assert torch.equal(loss.isnan(), bad)
    h.requires_grad_()
    g, = torch.autograd.grad(E.linear_distillation(h, w, index, t, reduction="none").sum(), h)
    assert torch.equal(g.isnan().any(1), bad)


def test_tokens_that_the_student_has_not():
    """A bias of -inf: an infinite loss where the teacher has the token, the others' losses as without it."""
    h, w, b, index, t = _inputs(30, 64, 100, 4, torch.float32, bias=torch.float32, holes=0.0)
    b[5] = -float("inf")
    index[index == 5] = 6
    index[3, 1] = 5
    index[2] = index[2].where(index[2] >= 0, 9)
    t[2, 1], index[2, 1] = -float("inf"), 5  # no entry
    want, bound = _reference(h, w, b, index, t, 1.0, "none")
    with torch.no_grad():
        got = E.linear_distillation(h, w, index, t, bias=b, reduction="none")
    assert bool(got[3].isinf()) and not bool(got[2].isinf())
    rest = torch.arange(30, device=DEV) != 3
    _close(got[rest], want[0][rest], bound[0][rest], "rows")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """int32 tokens, bfloat16 logits, the first of a longer list, turned ones, rows of three axes."""
    h, w, b, index, t = _inputs(24, 72, 300, 10, dtype, bias=dtype, logits=torch.bfloat16)
    base = _check(h, w, b, index[:, :6].contiguous(), t[:, :6].contiguous())
    for i, s in ((index[:, :6], t[:, :6]), (index[:, :6].int(), t[:, :6]),
                 (index[:, :6].t().contiguous().t(), t[:, :6].t().contiguous().t()), (index[:, :6], t[:, :6].float())):
        loss = E.linear_distillation(h, w, i, s, bias=b)
        assert torch.equal(loss, base[0])
    rows = E.linear_distillation(h.view(4, 6, 72), w, index.view(4, 6, 10), t.view(4, 6, 10), bias=b, reduction="none")
    assert rows.shape == (4, 6)
    assert torch.equal(rows.flatten(), E.linear_distillation(h, w, index, t, bias=b, reduction="none"))
    wide = torch.zeros(300, 80, device=DEV, dtype=dtype)
    wide[:, :72] = w
    assert torch.equal(E.linear_distillation(h, wide[:, :72], index[:, :6], t[:, :6], bias=b), base[0])


@pytest.mark.parametrize("N", [20, 400])
def test_kept_probabilities_and_new_ones_give_the_same_bits(N):
    h, w, b, index, t = _inputs(N, 64, 515, 9, torch.float32, bias=torch.float32)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    for reduction in ("none", "mean"):
        loss = E.linear_distillation(h, w, index, t, bias=b, temperature=2.0, reduction=reduction)
        up = torch.rand_like(loss) + 0.5
        first = torch.autograd.grad(loss, leaves, up, retain_graph=True)
        second = torch.autograd.grad(loss, leaves, up)
        for a, r in zip(first, second):
            assert torch.equal(a, r)


def test_gradient_against_differences():
    h, w, b, index, t = _inputs(20, 32, 70, 6, torch.float32, bias=torch.float32)
    leaves = [x.clone().requires_grad_() for x in (h, w, b)]
    loss = E.linear_distillation(*leaves[:2], index, t, bias=leaves[2], temperature=2.0, reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    step = 2.0**-6
    for k, g in enumerate(grads):
        way = torch.randn(g.shape, generator=torch.Generator(device=DEV).manual_seed(k), device=DEV)
        way /= way.norm()
        values = []
        for sign in (1, -1):
            x = [h, w, b]
            x[k] = x[k] + sign * step * way
            with torch.no_grad():
                values.append(E.linear_distillation(x[0], x[1], index, t, bias=x[2], temperature=2.0, reduction="none")
                              .double().sum())
        got, want = float((values[0] - values[1]) / (2 * step)), float((g.double() * way.double()).sum())
        # each row's loss is off by the reference's bound, 20 rows of some 2^-19 over 2^-5; the third derivative by
        # step^2 / 6 of a sum of 20 rows whose logits move by at most |h| step
        assert abs(got - want) <= 20 * 2.0**-19 / 2.0**-5 + step**2 / 6 * 20 * 32**1.5 * 0.05


def test_another_stream_and_the_same_bits():
    h, w, b, index, t = _inputs(300, 64, 2000, 40, torch.bfloat16, bias=torch.float32)
    want = _check(h, w, b, index, t)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        leaves = [x.clone().requires_grad_() for x in (h, w, b)]
        loss = E.linear_distillation(leaves[0], leaves[1], index, t, bias=leaves[2])
        got = (loss.detach(), *torch.autograd.grad(loss, leaves))
    side.synchronize()
    for a, r in zip(got, (want[0], *want[1])):
        assert torch.equal(a, r)


def test_scratch_holds_what_a_call_writes(monkeypatch):
    """The scratch between walls that have to stay as they are."""
    from ews_mi355x import loss as module

    walls = []
    plain = module._Call.workspace

    def walled(self, train):
        size = plain(self, train).numel()
        whole = torch.full((size + 8192,), 173, dtype=torch.uint8, device=DEV)
        walls.append((whole, size))
        return whole[4096:4096 + size]

    monkeypatch.setattr(module._Call, "workspace", walled)
    for N, H, V, K, dtype in ((1, 5, 3, 2, torch.float32), (33, 72, 700, 130, torch.bfloat16),
                              (300, 64, 2049, 1024, torch.float32), (700, 128, 1000, 7, torch.bfloat16)):
        for reduction in ("mean", "none"):
            _check(*_inputs(N, H, V, K, dtype, bias=dtype), reduction=reduction, planes=1)
    torch.cuda.synchronize()
    assert walls
    for whole, size in walls:
        assert bool((whole[:4096] == 173).all()) and bool((whole[4096 + size:] == 173).all())


def test_second_derivatives_are_refused():
    h, w, b, index, t = _inputs(8, 16, 30, 3, torch.float32)
    h.requires_grad_()
    g, = torch.autograd.grad(E.linear_distillation(h, w, index, t), h, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_no_rows():
    w = torch.randn(30, 16, device=DEV, requires_grad=True)
    h = torch.zeros(0, 16, device=DEV, requires_grad=True)
    index = torch.zeros(0, 3, dtype=torch.long, device=DEV)
    loss = E.linear_distillation(h, w, index, index.float())
    assert float(loss) == 0.0 and not torch.autograd.grad(loss, w)[0].any()
    assert E.linear_distillation(h, w, index, index.float(), reduction="none").shape == (0,)


def test_refusals_on_the_device():
    h, w, b, index, t = _inputs(8, 16, 30, 3, torch.float32)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        E.linear_distillation(h, w, index, t.half())
    with pytest.raises(TypeError, match="hidden is"):
        E.linear_distillation(h.bfloat16(), w, index, t)
    with pytest.raises(ValueError, match="indices are|indices is"):
        E.linear_distillation(h, w, index.cpu(), t)
    with pytest.raises(ValueError, match="detach"):
        E.linear_distillation(h, w, index, t.requires_grad_())
