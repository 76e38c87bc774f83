"""Gradient clipping (csrc/ews_clip.hip) against its formula. The norm is a float64 sum rounded once: it is within one
unit of float32. A clipped number is off by the coefficient's and its own rounding: two half units of float32 and half a
unit of its type."""

import math

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
HALF_UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def _tensors(shapes, dtypes, seed=0, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(s, generator=g, device=DEV) * size).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def _norm(tensors):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in tensors))


def _check(grads, max_norm, norm, outs):
    want = _norm(grads)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 2 * U * want
    c = min(1.0, max_norm / (want + 1e-6))
    for g, o in zip(grads, outs):
        r = g.double() * c
        assert o.dtype == g.dtype and o.shape == g.shape
        assert bool(((o.double() - r).abs() <= (4 * U + HALF_UNIT[g.dtype]) * r.abs() + 1e-38).all())


LISTS = [
    [(1,)],
    [(3, 5), (7,), (1, 1)],
    [(0,), (4, 4), (0, 3)],
    [(16384,), (16385,), (16383,), (3,)],
    [(100, 257), (64,), (1000, 33), (5,)],
    [(i % 37 + 1, i % 5 + 1) for i in range(300)],
    [(700, 1000), (2, 3), (1 << 20,)],
]


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("shapes", LISTS)
def test_clip(shapes, dtypes):
    grads = _tensors(shapes, dtypes)
    before = [g.clone() for g in grads]
    want = _norm(grads)
    for max_norm in (0.3 * want, 3.0 * want):
        norm, out = E.clip_grads(grads, max_norm)
        _check(grads, max_norm, norm, out)
        kept = [torch.full_like(g, float("nan")) for g in grads]
        norm2, out2 = E.clip_grads(grads, max_norm, out=kept)
        assert all(a is b for a, b in zip(out2, kept))
        assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(out, kept))
        if max_norm > want:
            assert all(torch.equal(a, b) for a, b in zip(out, grads))
        params = [torch.zeros_like(g).requires_grad_() for g in grads]
        params.append(torch.zeros(3, device=DEV, requires_grad=True))
        for p, g in zip(params, grads):
            p.grad = g.clone()
        norm3 = E.clip_grad_norm_(params, max_norm)
        assert torch.equal(norm, norm3) and all(torch.equal(p.grad, o) for p, o in zip(params, out))
        assert params[-1].grad is None
    assert torch.equal(E.global_grad_norm(grads), norm)
    assert all(torch.equal(a, b) for a, b in zip(before, grads))


def test_sizes_out_of_float32_range():
    """Squares that float32 does not hold, above and below."""
    for size in (1e25, 1e-25):
        grads = _tensors([(5000,), (33, 3)], [torch.float32], size=size)
        assert abs(float(E.global_grad_norm(grads)) / _norm(grads) - 1.0) <= 2 * U
    norm, out = E.clip_grads(_tensors([(5000,)], [torch.float32], size=1e25), 1.0)
    assert abs(_norm(out) - 1.0) < 1e-5


def test_not_finite():
    grads = _tensors([(100,), (50, 2)], [torch.float32])
    grads[0][7] = float("inf")
    norm, out = E.clip_grads(grads, 1.0)
    assert float(norm) == float("inf") and not bool(out[1].any()) and bool(torch.isnan(out[0][7]))
    grads[1][3, 1] = float("nan")
    norm, out = E.clip_grads(grads, 1.0)
    assert bool(torch.isnan(norm)) and all(bool(torch.isnan(o).all()) for o in out)
    zeros = [torch.zeros(40, device=DEV)]
    norm, out = E.clip_grads(zeros, 0.0)
    assert float(norm) == 0.0 and not bool(out[0].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    base = torch.randn(70, 90, device=DEV).to(dtype)
    flat = torch.randn(40001, device=DEV).to(dtype)
    views = [base.t(), base[::2, 1:50], base[3], base[:, 7], flat[1:20000], flat[20001:40000],
             base[:3, :1].expand(3, 4)]
    norm, out = E.clip_grads(views, 1.0)
    _check([v.clone() for v in views], 1.0, norm, out)
    # in place through every view of which no two elements share memory
    copies = [base.clone().t(), base.clone()[::2, 1:50], base.clone()[:, 7], flat.clone()[1:20000]]
    before = [c.clone() for c in copies]
    norm, out = E.clip_grads(copies, 1.0, out=copies)
    _check(before, 1.0, norm, copies)
    # out with other strides than the gradient's
    other = [torch.empty(90, 70, device=DEV, dtype=dtype).t()]
    norm, _ = E.clip_grads([base], 1.0, out=other)
    _check([base], 1.0, norm, other)


def test_none_and_streams():
    assert float(E.global_grad_norm([])) == 0.0
    assert float(E.clip_grad_norm_([], 1.0)) == 0.0
    assert E.clip_grads([], 1.0)[1] == []
    grads = _tensors([(300, 300), (17,)], [torch.float32])
    want = E.clip_grads(grads, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = E.clip_grads(grads, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want[0], got[0]) and all(torch.equal(a, b) for a, b in zip(want[1], got[1]))


def test_refusals_on_the_device():
    g = torch.ones(4, device=DEV)
    for call, kind in ((lambda: E.clip_grads([g], -1.0), ValueError),
                       (lambda: E.clip_grads([g], float("nan")), ValueError),
                       (lambda: E.clip_grads([g.double()], 1.0), TypeError),
                       (lambda: E.clip_grads([g.cpu()], 1.0), RuntimeError),
                       (lambda: E.clip_grads([g], 1.0, out=[]), ValueError),
                       (lambda: E.clip_grads([g], 1.0, out=[g[:3]]), ValueError),
                       (lambda: E.clip_grads([g], 1.0, out=[g.bfloat16()]), ValueError),
                       (lambda: E.global_grad_norm([g.to_sparse()]), TypeError)):
        with pytest.raises(kind):
            call()


def test_a_parameter_named_twice_counts_once():
    (g,) = _tensors([(70, 33)], [torch.float32])
    p = torch.zeros_like(g).requires_grad_()
    p.grad = g.clone()
    norm = E.clip_grad_norm_([p, p], 0.5)
    _check([g], 0.5, norm, [p.grad])
