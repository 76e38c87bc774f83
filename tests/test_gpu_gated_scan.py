"""``gated_scan`` on the device against the recurrence step by step in float64: every kernel (threads that walk alone,
tiles of 64 and 32 lanes and narrower ones, segments), types, forms, masks, states, strides."""

import pytest
import torch

from scan_oracle import assert_near, recurrence

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def _inputs(B, L, D, dtype, form, seed=0, state=True, mask=None):
    g = torch.Generator().manual_seed(1000 * seed + 31 * B + 7 * L + D)
    x = torch.randn(B, L, D, generator=g).to(dtype)
    gate = torch.randn(B, L, D, generator=g) * 2 + 1
    gate = (gate if form == "convex" else torch.sigmoid(gate)).to(dtype)
    s = torch.randn(B, D, generator=g) if state else None
    m = None
    if mask == "tail":
        m = torch.arange(L)[None] < torch.randint(0, L + 1, (B, 1), generator=g)
    elif mask == "holes":
        m = torch.rand(B, L, generator=g) < 0.7
    elif mask == "none":
        m = torch.zeros(B, L, dtype=torch.bool)
    return x, gate, s, m, torch.randn(B, L, D, generator=g).to(dtype), torch.randn(B, D, generator=g)


def _check(x, gate, state, mask, form, dh, dlast, forward_only=False):
    import ews_mi355x as E

    want = recurrence(x.double(), gate.double(), None if state is None else state.double(), mask, form, dh.double(),
                      dlast.double())
    dev = [None if t is None else t.cuda() for t in (x, gate, state)]
    m = None if mask is None else mask.cuda()
    with torch.no_grad():
        h, last = E.gated_scan(*dev, mask=m, form=form)
    assert h.dtype is x.dtype and last.dtype is torch.float32
    assert_near(h, *want["h"], "h")
    assert_near(last, *want["last"], "last")
    if forward_only:
        return
    leaves = [None if t is None else t.clone().requires_grad_() for t in dev]
    h2, last2 = E.gated_scan(*leaves, mask=m, form=form)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    grads = torch.autograd.grad((h2, last2), [t for t in leaves if t is not None], (dh.cuda(), dlast.cuda()))
    for name, g in zip(("dx", "dgate", "dstate"), grads):
        assert_near(g, *want[name], name)


@pytest.mark.parametrize("form", ["convex", "linear"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,D", [
    (1, 1, 1), (8, 1, 2048), (3, 2, 5), (2, 16, 70), (2, 17, 70), (1, 17, 1), (2, 129, 8), (3, 200, 9), (2, 257, 16),
    (1, 300, 24), (2, 127, 33), (2, 128, 64), (1, 513, 130),
    (600, 17, 450),    # alone: 4800 wavefronts of float32
    (1100, 18, 500),   # alone in bfloat16 pairs too
    (128, 40, 516),    # 64 lanes
    (12, 260, 516),    # 32 lanes of float32
    (24, 260, 516),    # 32 lanes of bfloat16 pairs
    (1, 2100, 3),      # segments
    (2, 4099, 40),
])
def test_sizes(B, L, D, dtype, form):
    _check(*_args(_inputs(B, L, D, dtype, form), form))


def _args(inputs, form):
    x, gate, state, mask, dh, dlast = inputs
    return x, gate, state, mask, form, dh, dlast


@pytest.mark.parametrize("mask", ["tail", "holes", "none"])
@pytest.mark.parametrize("form", ["convex", "linear"])
@pytest.mark.parametrize("B,L,D", [(3, 9, 70), (2, 130, 24), (2, 2050, 12), (600, 20, 450)])
def test_masks(B, L, D, form, mask):
    x, gate, state, m, dh, dlast = _inputs(B, L, D, torch.float32, form, mask=mask)
    _check(x, gate, state, m, form, dh, dlast)
    # what masked steps hold is not used
    import ews_mi355x as E

    bad_x, bad_g = x.clone(), gate.clone()
    bad_x[~m], bad_g[~m] = float("nan"), float("inf")
    good = [t.cuda().requires_grad_() for t in (x, gate, state)]
    bad = [t.cuda().requires_grad_() for t in (bad_x, bad_g, state)]
    outs = []
    for leaves in (good, bad):
        h, last = E.gated_scan(*leaves, mask=m.cuda(), form=form)
        outs.append((h, last, *torch.autograd.grad((h, last), leaves, (dh.cuda(), dlast.cuda()))))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    off = ~m.cuda()
    assert not outs[0][2][off].any() and not outs[0][3][off].any()


def test_one_mask_for_all_sequences():
    import ews_mi355x as E

    x, gate, state, _, _, _ = (None if t is None else t.cuda() for t in _inputs(3, 50, 20, torch.float32, "convex"))
    m = torch.arange(50, device="cuda") % 3 != 0
    assert torch.equal(E.gated_scan(x, gate, mask=m)[0], E.gated_scan(x, gate, mask=m.expand(3, 50).contiguous())[0])
    turned = m[:, None].expand(50, 3).contiguous().t()
    assert torch.equal(E.gated_scan(x, gate, mask=m)[0], E.gated_scan(x, gate, mask=turned)[0])


@pytest.mark.parametrize("L", [300, 2100])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype, L):
    """The halves of a joint projection, a transposed batch, rows off 4-byte addresses: read where they are."""
    import ews_mi355x as E

    both = torch.randn(2, L, 48, device="cuda").to(dtype)
    x, gate = both.chunk(2, -1)
    want = E.gated_scan(x.contiguous(), gate.contiguous())
    for a, b in zip(E.gated_scan(x, gate), want):
        assert torch.equal(a, b)
    flipped = both.transpose(0, 1).contiguous().transpose(0, 1)
    for a, b in zip(E.gated_scan(*flipped.chunk(2, -1)), want):
        assert torch.equal(a, b)
    last_first = both.transpose(1, 2).contiguous().transpose(1, 2)
    for a, b in zip(E.gated_scan(*last_first.chunk(2, -1)), want):
        assert torch.equal(a, b)
    odd = torch.empty(2 * L * 24 + 1, device="cuda", dtype=dtype)[1:].view(2, L, 24)
    odd.copy_(x)
    for a, b in zip(E.gated_scan(odd, gate), want):
        torch.testing.assert_close(a, b, rtol=0, atol=0)
    # and their gradients, the upstream one off its address too
    u = torch.empty(2 * L * 24 + 1, device="cuda", dtype=dtype)[1:].view(2, L, 24).normal_()
    joint = both.clone().requires_grad_()
    h, _ = E.gated_scan(*joint.chunk(2, -1))
    apart = [t.contiguous().detach().requires_grad_() for t in (x, gate)]
    h2, _ = E.gated_scan(*apart)
    got = torch.autograd.grad(h, joint, u)[0]
    want = torch.cat(torch.autograd.grad(h2, apart, u.clone()), -1)
    assert torch.equal(got, want)


@pytest.mark.parametrize("which", ["h", "last"])
@pytest.mark.parametrize("L", [1, 40, 2100])
def test_one_output_alone(L, which):
    import ews_mi355x as E

    x, gate, state, _, dh, dlast = _inputs(2, L, 24, torch.float32, "convex")
    zero = torch.zeros_like(dh) if which == "last" else torch.zeros_like(dlast)
    want = recurrence(x.double(), gate.double(), state.double(), None, "convex",
                      dh.double() if which == "h" else zero.double(), dlast.double() if which == "last" else zero.double())
    leaves = [t.cuda().requires_grad_() for t in (x, gate, state)]
    h, last = E.gated_scan(*leaves)
    grads = torch.autograd.grad(h if which == "h" else last, leaves, (dh if which == "h" else dlast).cuda())
    for name, g in zip(("dx", "dgate", "dstate"), grads):
        assert_near(g, *want[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_that_are_shut_or_open(dtype):
    """A gate of -inf takes the step's input alone, one of +inf keeps the state; far gates do not overflow."""
    import ews_mi355x as E

    x = torch.randn(1, 40, 6).to(dtype).cuda()
    gate = torch.zeros(1, 40, 6, device="cuda", dtype=dtype)
    for value, want in ((-float("inf"), x), (-1e30, x), (-90.0, x)):
        got, _ = E.gated_scan(x, gate + value)
        torch.testing.assert_close(got, want, rtol=2.0**-23, atol=1e-35)
    state = torch.randn(1, 6, device="cuda")
    for value in (float("inf"), 1e30, 200.0):
        _, last = E.gated_scan(x, gate + value, state=state)
        assert torch.equal(last, state)
    broken = gate.clone()
    broken[0, 7, 2] = float("nan")
    h, last = E.gated_scan(x, broken)
    assert bool(h[0, 7:, 2].isnan().all()) and not bool(h[0, :7].isnan().any()) and bool(last[0, 2].isnan())
    assert int(h.isnan().sum()) == 33


@pytest.mark.parametrize("L,cuts", [(64, (1, 2, 3, 30, 63)), (2100, (8, 1000, 1999))])
def test_parts_with_their_states(L, cuts):
    """A sequence in parts, each from the state that the one before handed back, a single token among them."""
    import ews_mi355x as E

    x, gate, state, _, _, _ = _inputs(2, L, 24, torch.float32, "convex")
    want = recurrence(x.double(), gate.double(), state.double(), None, "convex", torch.zeros(2, L, 24).double(), None)
    s, at, rows = state.cuda(), 0, []
    for end in (*cuts, L):
        h, s = E.gated_scan(x[:, at:end].cuda(), gate[:, at:end].cuda(), state=s)
        rows.append(h)
        at = end
    # a state that is handed back is rounded as it would be within the sequence
    assert_near(torch.cat(rows, 1), *want["h"])
    assert_near(s, *want["last"])


@pytest.mark.parametrize("L", [1, 5, 300, 2100])
def test_last_in_place(L):
    import ews_mi355x as E

    x, gate, state, _, _, _ = (None if t is None else t.cuda() for t in _inputs(2, L, 24, torch.float32, "convex"))
    h, want = E.gated_scan(x, gate, state=state)
    s = state.clone()
    h2, got = E.gated_scan(x, gate, state=s, last=s)
    assert got is s and torch.equal(s, want) and torch.equal(h, h2)
    other = torch.empty_like(s)
    assert E.gated_scan(x, gate, state=state, last=other)[1] is other and torch.equal(other, want)


def test_empty():
    import ews_mi355x as E

    state = torch.randn(2, 5, device="cuda", requires_grad=True)
    x = torch.zeros(2, 0, 5, device="cuda", requires_grad=True)
    h, last = E.gated_scan(x, x.detach(), state=state)
    assert h.shape == (2, 0, 5) and torch.equal(last, state)
    assert torch.autograd.grad(last.sum() + h.sum(), [x, state])[1].eq(1).all()
    h, last = E.gated_scan(torch.zeros(0, 4, 5, device="cuda"), torch.zeros(0, 4, 5, device="cuda"))
    assert h.shape == (0, 4, 5) and last.shape == (0, 5)
    none = torch.zeros(2, 0, 5, device="cuda")
    assert not E.gated_scan(none, none)[1].any()


@pytest.mark.parametrize("form", ["convex", "linear"])
def test_gradients_against_differences(form):
    """Central differences of a float64 sum of the outputs, along random directions."""
    import ews_mi355x as E

    x, gate, state, mask, dh, dlast = (t.cuda() for t in _inputs(2, 150, 10, torch.float32, form, mask="holes"))
    leaves = [t.clone().requires_grad_() for t in (x, gate, state)]
    h, last = E.gated_scan(*leaves, mask=mask, form=form)
    grads = torch.autograd.grad((h, last), leaves, (dh, dlast))

    def value(*inputs):
        with torch.no_grad():
            h, last = E.gated_scan(*inputs, mask=mask, form=form)
        return float((h.double() * dh.double()).sum() + (last.double() * dlast.double()).sum())

    step = 2.0**-8
    for k, g in enumerate(grads):
        way = torch.randn(g.shape, generator=torch.Generator().manual_seed(k)).cuda()
        up, down = [x, gate, state], [x, gate, state]
        up[k], down[k] = up[k] + step * way, down[k] - step * way
        got = (value(*up) - value(*down)) / (2 * step)
        want = float((g.double() * way.double()).sum())
        # the difference's own error: step^2 / 6 of the third derivative along a direction of length sqrt(n), and the
        # float32 rounding of 3000 terms over 2 step: both under 1e-3 of the gradient's length
        assert abs(got - want) <= 1e-3 * float(g.double().norm()) * 10
