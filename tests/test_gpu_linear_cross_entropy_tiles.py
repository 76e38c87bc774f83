"""Linear cross entropy (csrc/ews_loss.hip) on each of its tiles, in chunks, and through its entry points' two halves,
against the formula in float64.

Bounds, number by number, with u = 2^-24, half(T) = 2^-24 or 2^-8 (the relative error of one rounding to T) and S =
sum_k |h_k w_k|: a logit is off by at most (H + 8) u S, a loss by twice that and 8 u (1 + |z|) and, for the slabs joined
one after another, 200 u. A probability is off by the factor e = 2 max (H + 8) u S + 16 u + 2 u max |z|, and where it is
kept as a 16-bit logarithm in steps of 1/512 octave by 2^-10.5 more. dz carries that and its own rounding:
half(bfloat16) |dz| in one bfloat16, half(bfloat16)^2 in two. A gradient is off by dz's error times the other operand's
magnitude, its float32 sum's (K + 8) u of the summed magnitudes, half of its own type and 2 u of the mean's factor."""

import ctypes
import math

import pytest
import torch

import ews_mi355x as E
from ews_mi355x import _native as nat
from loss_shapes import TILES

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _inputs(N, H, V, dtype, seed=0):
    """Rows that lean towards their target's row of the weight; every seventh row ignored."""
    g = torch.Generator(device=DEV).manual_seed(seed + N + 31 * H + 7 * V)
    w = (torch.randn(V, H, generator=g, device=DEV) * (1.5 / math.sqrt(H))).to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device=DEV)
    t[0], t[N - 1] = V - 1, 0  # the last columns' remainder holds a target
    h = (torch.randn(N, H, generator=g, device=DEV) + 3.0 * torch.rand(N, 1, generator=g, device=DEV) * w[t]).to(dtype)
    b = 0.5 * torch.randn(V, generator=g, device=DEV)
    up = torch.rand(N, generator=g, device=DEV) + 0.5
    t[3::7] = -100
    return h, w, b, t, up


def _two_planes(dtype, N, reduction):
    return dtype == torch.bfloat16 and N <= (256 if reduction == "none" else 16)


def _reference(h, w, b, t, up, reduction, step=256):
    """((loss, bound), ...) of the loss and the three gradients, kept rows in steps."""
    N, H = h.shape
    V = w.shape[0]
    keep = (t != -100).nonzero()[:, 0]
    scale = 1.0 / max(1, len(keep)) if reduction == "mean" else 1.0
    wd, bd = w.double(), b.double()
    loss, lerr = (torch.zeros(N, device=DEV, dtype=torch.float64) for _ in range(2))
    gh, herr = (torch.zeros(N, H, device=DEV, dtype=torch.float64) for _ in range(2))
    gw, werr = (torch.zeros(V, H, device=DEV, dtype=torch.float64) for _ in range(2))
    gb, berr = (torch.zeros(V, device=DEV, dtype=torch.float64) for _ in range(2))
    half = HALF[h.dtype]
    for rows in keep.split(step):
        x, tk, at = h[rows].double(), t[rows], torch.arange(len(rows), device=DEV)
        z = torch.addmm(bd, x, wd.t())
        zerr = (H + 8) * U * (x.abs() @ wd.abs().t()).max(1).values
        zmag = z.abs().max(1).values
        loss[rows] = torch.logsumexp(z, 1) - z[at, tk]
        lerr[rows] = 2 * zerr + 8 * U * (1 + zmag) + 200 * U
        p = torch.softmax(z, 1)
        g = (up[rows].double() if reduction == "none" else torch.full_like(zmag, scale))[:, None]
        e = (2 * zerr + 16 * U + 2 * U * zmag)[:, None]
        if h.dtype == torch.bfloat16:
            e = e + 1.1 * 2.0**-10.5
        derr = p * e * g
        d = p
        d[at, tk] -= 1.0
        d *= g
        own = 4 * U if h.dtype == torch.float32 else half * half if _two_planes(h.dtype, N, reduction) else 1.01 * half
        derr += own * d.abs()
        gh[rows] = d @ wd
        herr[rows] = derr @ wd.abs() + (V + 8) * U * (d.abs() @ wd.abs())
        gw += d.t() @ x
        werr += derr.t() @ x.abs() + (len(keep) + 8) * U * (d.abs().t() @ x.abs())
        gb += d.sum(0)
        berr += derr.sum(0) + (len(keep) + 8) * U * d.abs().sum(0)
    if reduction != "none":
        loss, lerr = loss.sum() * scale, lerr.sum() * scale
        lerr = lerr + U * loss.abs()
    return ((loss, lerr), (gh, herr + (half + 2 * U) * gh.abs()), (gw, werr + (half + 2 * U) * gw.abs()),
            (gb, berr + 3 * U * gb.abs()))


def _close(got, want, bound, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    ok = err <= bound + 1e-36  # NaN is not
    assert bool(ok.all()), (what, float((err / (bound + 1e-36)).max()), int((~ok).sum()))


def _check(h, w, b, t, up, reduction, score=True):
    wrt = [x.detach().requires_grad_() for x in (h, w, b)]
    loss = E.linear_cross_entropy(wrt[0], wrt[1], t, bias=wrt[2], reduction=reduction)
    got = torch.autograd.grad(loss, wrt, up if reduction == "none" else None)
    want = _reference(h, w, b, t, up, reduction)
    for name, a, (r, e) in zip(("loss", "grad_hidden", "grad_weight", "grad_bias"), (loss.detach(), *got), want):
        _close(a, r, e, name)
    assert not bool(got[0][3::7].any())
    if score:
        with torch.no_grad():
            _close(E.linear_cross_entropy(h, w, t, bias=b, reduction=reduction), *want[0], "score")


@pytest.mark.parametrize("key", TILES, ids=str)
def test_tiles(key):
    print(f"loss on {TILES[key]}: {key}", flush=True)
    dtype, N, H, V, reduction = key
    _check(*_inputs(N, H, V, getattr(torch, dtype)), reduction)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unaligned_weight_and_strides_on_the_large_tile(dtype):
    N, H, V = 1030, 776, 9001
    h, w, b, t, up = _inputs(N, H, V, dtype)
    wide = torch.zeros(V, H + 9, device=DEV, dtype=dtype)
    wide[:, 3:H + 3] = w
    tall = torch.zeros(N, H + 5, device=DEV, dtype=dtype)
    tall[:, 1:H + 1] = h
    print(f"strided {dtype}", flush=True)
    _check(tall[:, 1:H + 1], wide[:, 3:H + 3], b, t, up, "mean", score=False)


@pytest.mark.parametrize("dtype,N,reduction", [(torch.float32, 1100, "none"), (torch.bfloat16, 5000, "none"),
                                               (torch.bfloat16, 5000, "mean")])
def test_chunks(dtype, N, reduction):
    """More rows than are kept at a time, so the rows' own losses are computed again by the backward, and dW is summed
    over the chunks; the loss of the second backward is the first's."""
    V, H = 300007, 72
    print(f"chunks {dtype} N={N} {reduction}", flush=True)
    h, w, b, t, up = _inputs(N, H, V, dtype)
    desc = nat.LossDesc(hidden_stride=H, weight_stride=H, ignore_index=-100, rows=N, hidden=H, vocab=V,
                        dtype=0 if dtype == torch.float32 else 1, bias_dtype=0,
                        reduction=nat.LOSS_REDUCTIONS[reduction])
    tile = (ctypes.c_int32 * 4)()
    assert nat.load().ews_loss_tile(desc, w.data_ptr(), 1, 0, tile) == 0 and tile[3] > 1
    assert not nat.load().ews_loss_keeps(desc)
    _check(h, w, b, t, up, reduction, score=False)
    t[N // 4:] = -100  # later chunks hold nothing
    h, w, b = (x.requires_grad_() for x in (h, w, b))
    loss = E.linear_cross_entropy(h, w, t, bias=b, reduction=reduction)
    got = torch.autograd.grad(loss, [h, w, b], up if reduction == "none" else None)
    want = _reference(h.detach(), w.detach(), b.detach(), t, up, reduction)
    for name, a, (r, e) in zip(("loss", "grad_hidden", "grad_weight", "grad_bias"), (loss.detach(), *got), want):
        _close(a, r, e, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [9, 300])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_the_two_halves_give_the_whole(reduction, N, dtype):
    """ews_loss_keep and ews_loss_kept as the C ABI has them, for every reduction, against ews_loss_train."""
    H, V = 136, 700
    h, w, b, t, up = _inputs(N, H, V, dtype)
    lib = nat.load()
    desc = nat.LossDesc(hidden_stride=H, weight_stride=H, ignore_index=-100, rows=N, hidden=H, vocab=V,
                        dtype=0 if dtype == torch.float32 else 1, bias_dtype=0,
                        reduction=nat.LOSS_REDUCTIONS[reduction])
    assert lib.ews_loss_keeps(desc) == 1
    size = lib.ews_loss_workspace_bytes_for(desc, w.data_ptr(), 1)
    st = torch.cuda.current_stream().cuda_stream
    upstream = up.data_ptr() if reduction == "none" else None

    def buffers():
        return (torch.empty(N if reduction == "none" else 1, device=DEV), torch.empty_like(h), torch.empty_like(w),
                torch.empty_like(b), torch.empty(size, dtype=torch.uint8, device=DEV))

    loss, gh, gw, gb, ws = one = buffers()
    inputs = (h.data_ptr(), w.data_ptr(), b.data_ptr(), t.data_ptr())
    assert lib.ews_loss_train(desc, *inputs, upstream, loss.data_ptr(), gh.data_ptr(), gw.data_ptr(), gb.data_ptr(),
                              ws.data_ptr(), st) == 0
    loss, gh, gw, gb, ws = two = buffers()
    assert lib.ews_loss_keep(desc, *inputs, loss.data_ptr(), gh.data_ptr(), ws.data_ptr(), st) == 0
    assert lib.ews_loss_kept(desc, w.data_ptr(), upstream, gh.data_ptr(), gw.data_ptr(), gb.data_ptr(), ws.data_ptr(),
                             st) == 0
    for a, c in zip(one[:4], two[:4]):
        assert torch.equal(a, c)
    want = _reference(h, w, b, t, up, reduction)
    for name, a, (r, e) in zip(("loss", "grad_hidden", "grad_weight", "grad_bias"), one, want):
        _close(a.reshape(r.shape), r, e, name)


@pytest.mark.parametrize("reduction,N,V", [("mean", 300, 1003), ("none", 300, 1003), ("sum", 1030, 9001)])
def test_dz_number_by_number(reduction, N, V):
    """Row n of h is 3 in column n alone, so a number of dW is 3 dz of one row: dz's errors do not average out. One
    rounding of dz to bfloat16, one of the result and the logarithm's steps are allowed; probabilities held in bfloat16
    would add a rounding."""
    H = N
    _, w, b, t, up = _inputs(N, H, V, torch.bfloat16)
    w = (w.float() * math.sqrt(H)).bfloat16()  # logits of a few units
    h = torch.zeros(N, H, device=DEV, dtype=torch.bfloat16).fill_diagonal_(3.0).requires_grad_()
    w.requires_grad_()
    loss = E.linear_cross_entropy(h, w, t, bias=b, reduction=reduction)
    (gw,) = torch.autograd.grad(loss, [w], up if reduction == "none" else None)
    z = 3.0 * w.detach().double().t() + b.double()
    d = torch.softmax(z, 1)
    kept = (t != -100).nonzero()[:, 0]
    d[kept, t[kept]] -= 1.0
    d *= (t != -100)[:, None]
    d *= (up.double() if reduction == "none" else torch.full_like(z[:, 0], 1.0 / len(kept)) if reduction == "mean"
          else torch.ones_like(z[:, 0]))[:, None]
    want = 3.0 * d.t()
    half = 2.0**-8
    f32 = 16 * U + 8 * U * (1 + float(z.abs().max()))  # the logits', the sums' and the factors' roundings
    bound = (1.01 * half + half + 1.1 * 2.0**-10.5 + f32) * want.abs()
    own = torch.zeros_like(bound)
    own[t[kept], kept] = 3.0 * f32  # the targets' entries: p - 1 of a p that is off by f32
    _close(gw, want, bound + own, "dW")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_an_upstream_number_multiplies_the_rounded_gradients(reduction, dtype):
    """Of the mean and the sum: a power of two rounds nothing, another number once more, and the upstream numbers of a
    sum of losses are each their own."""
    h, w, b, t, _ = _inputs(300, 72, 515, dtype)
    wrt = [x.requires_grad_() for x in (h, w, b.to(dtype))]

    def grads(factor):
        loss = E.linear_cross_entropy(wrt[0], wrt[1], t, bias=wrt[2], reduction=reduction)
        return torch.autograd.grad(loss * factor, wrt)

    one = grads(1.0)
    for factor in (0.25, -2.0, 3.0, 0.3, 0.0):
        scale = torch.tensor(factor, device=DEV)
        for a, c in zip(grads(factor), one):
            assert torch.equal(a, (c.float() * scale).to(dtype))
    two = [E.linear_cross_entropy(wrt[0], wrt[1], t, bias=wrt[2], reduction=reduction) for _ in range(2)]
    got = torch.autograd.grad(two[0] * 3.0 + two[1] * 0.3, wrt)
    for a, x, y in zip(got, grads(3.0), grads(0.3)):
        assert torch.equal(a, x + y)
