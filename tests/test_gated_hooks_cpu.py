"""What the backward calls of ``gated_scan`` and ``gated_linear`` hand to the library where hooks on saved tensors bring
them back with other strides or at other addresses: descriptors and scratch of the tensors that came back. The launches
are recorded, not run."""

import ctypes

import pytest
import torch

from ews_mi355x import _native as nat
from ews_mi355x import gated, recurrence


def _value(a):
    return a.value if isinstance(a, ctypes.c_void_p) else a


@pytest.fixture
def calls(monkeypatch):
    made = []

    def record(dev, fn, *args):
        made.append((fn.__name__, [_value(a) for a in args]))
        return 0

    monkeypatch.setattr(recurrence, "launch", record)
    monkeypatch.setattr(gated, "launch", record)
    return made


class _Elsewhere:
    """Hooks that bring saved tensors back contiguous, ``off`` bytes behind a multiple of 64."""

    def __init__(self, off=0):
        self.off, self.came = off, {}

    def unpack(self, t):
        size = t.element_size()
        flat = torch.empty(t.numel() * size + 192, dtype=torch.uint8)
        flat = flat[-flat.data_ptr() % 64 + self.off:][:t.numel() * size].view(t.dtype).view(t.shape)
        flat.copy_(t)
        self.came[flat.data_ptr()] = flat
        return flat

    def __enter__(self):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t, self.unpack)
        self.hooks.__enter__()
        return self

    def __exit__(self, *args):
        self.hooks.__exit__(*args)


def _halves(B, L, D, dtype):
    joint = torch.randn(B, L, 2 * D).to(dtype).requires_grad_()
    return joint, joint.chunk(2, -1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
def test_scan_backward_describes_what_came_back(calls, dtype, masked):
    _, (x, gate) = _halves(2, 30, 24, dtype)
    mask = (torch.arange(30) % 3 != 0).expand(2, 30) if masked else None
    with _Elsewhere() as there:
        h, last = recurrence._GatedScan.apply(x, gate, None, mask, "convex")
    (h.float().sum() + last.sum()).backward()
    (_, forward), (name, (desc, px, pg, pm, *_)) = calls
    assert name == "ews_gated_scan_backward" and (forward[0].x_batch, forward[0].x_step) == (30 * 48, 48)
    for p, stride in ((px, (desc.x_batch, desc.x_step)), (pg, (desc.gate_batch, desc.gate_step))):
        assert there.came[p].stride() == (*stride, 1)
    if masked:
        assert there.came[pm].stride(0) == desc.mask_batch


def test_scan_backward_without_hooks_reads_where_the_forward_did(calls):
    _, (x, gate) = _halves(2, 30, 24, torch.float32)
    h, _ = recurrence._GatedScan.apply(x, gate, None, None, "convex")
    h.sum().backward()
    (_, f), (_, b) = calls
    assert b[0] is f[0] and b[1:3] == f[1:3]


def test_scan_refuses_a_saved_tensor_of_another_type_or_shape(calls):
    for change, says in ((lambda t: t.double() if t.is_floating_point() else t, "came back as torch.float64"),
                         (lambda t: t[..., :3].contiguous() if t.dim() == 3 else t, r"\(2, 30, 3\)")):
        _, (x, gate) = _halves(2, 30, 24, torch.float32)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            h, _ = recurrence._GatedScan.apply(x, gate, None, None, "convex")
        with pytest.raises(RuntimeError, match=says):
            h.sum().backward()
    assert all(name != "ews_gated_scan_backward" for name, _ in calls)


@pytest.mark.parametrize("B,L,D", [(1, 17, 2), (2, 200, 24), (8, 4095, 2048), (1, 131071, 1024), (600, 17, 450)])
def test_the_residual_does_not_depend_on_strides(B, L, D):
    """The tiles whose first states a forward leaves are those that its backward looks for."""
    lib = nat.load()
    sizes = set()
    for step in (D, 2 * D, 2 * D + 1):
        d = nat.GatedScanDesc(L * step, step, L * D, D, L, B, L, D, nat.DTYPE_BF16, 0)
        sizes.add((lib.ews_gated_scan_residual_bytes(d), lib.ews_gated_scan_workspace_bytes(d)))
    assert len(sizes) == 1


def _apart(rows, cols, stride, dtype):
    return torch.randn(rows, stride).to(dtype)[:, :cols].requires_grad_()


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("dtype,off", [(torch.float32, 0), (torch.float32, 4), (torch.bfloat16, 0), (torch.bfloat16, 2),
                                       (torch.bfloat16, 4)])
def test_gated_backward_describes_what_came_back(calls, monkeypatch, dtype, off, joint):
    """Strides, V's and G's addresses, and scratch as large as the plan of these addresses asks for."""
    N, H, F, sizes = 100, 128, 96, []
    scratch = gated._scratch

    def seen(x, size):
        sizes.append(size)
        return scratch(x, size)

    monkeypatch.setattr(gated, "_scratch", seen)
    x, w = _apart(N, H, 136, dtype), _apart(2 * F if joint else F, H, 144, dtype)
    g = None if joint else _apart(F, H, 144, dtype)
    with _Elsewhere(off) as there:
        y = gated._GatedLinear.apply(x, w, None, g, None, "silu")
    y.float().sum().backward()
    (_, forward), (name, (desc, px, pv, _, pg, _, kept, *_)) = calls
    assert name == "ews_gated_backward" and forward[0].x_stride == 136 and forward[0].weight_stride == 144
    came = there.came
    assert (desc.x_stride, desc.weight_stride, desc.gate_stride) == (H, H, H)
    assert came[px].shape == (N, H) and came[pv].shape == w.shape
    assert pg == pv + F * H * w.element_size() if joint else came[pg].shape == (F, H)
    assert kept % 16 == 0
    assert sizes[-1] >= nat.load().ews_gated_workspace_bytes(desc, px, pv, pg, nat.GATED_BACKWARD) > 0


def test_gated_backward_without_hooks_reads_where_the_forward_did(calls):
    y = gated._GatedLinear.apply(_apart(100, 128, 136, torch.float32), _apart(192, 128, 128, torch.float32), None, None,
                                 None, "silu")
    y.sum().backward()
    (_, f), (_, b) = calls
    assert b[0] is f[0] and b[1:6] == f[1:6]


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("turned", [False, True])
def test_a_stages_graph_of_its_backward(calls, joint, turned):
    """Its gradients and theirs are those of the maps; turned weights, which the library copies, keep theirs."""
    N, H, F = 9, 6, 5
    g = torch.Generator().manual_seed(1)

    def leaf(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float32).requires_grad_()

    x, up = leaf(N, H), leaf(N, F)
    w, b = leaf(*((H, 2 * F if joint else F) if turned else (2 * F if joint else F, H))), leaf(2 * F if joint else F)
    gw, gb = (None, None) if joint else (leaf(F, H), leaf(F))
    leaves = [t for t in (x, w, b, gw, gb) if t is not None]
    first = []
    for fused in (True, False):
        weight = w.t() if turned else w
        if fused:
            y = gated._GatedStage.apply(x, weight, b, gw, gb, "sigmoid")
        else:
            z = torch.nn.functional.linear(x, weight, b)
            v, s = z.chunk(2, -1) if joint else (z, torch.nn.functional.linear(x, gw, gb))
            y = v * torch.sigmoid(s)
        grads = torch.autograd.grad(y, leaves, up, create_graph=True)
        first.append((grads, torch.autograd.grad(sum(t.square().sum() for t in grads), [*leaves, up])))
    for (a, a2), (r, r2) in [first]:
        for s, t in zip((*a, *a2), (*r, *r2)):
            assert torch.equal(s, t)
    assert [name for name, _ in calls] == ["ews_gated_forward"]


def test_a_stages_backward_of_many_gradients_at_a_time(calls):
    g = torch.Generator().manual_seed(2)
    x, w, b = (torch.randn(*s, generator=g).requires_grad_() for s in ((9, 6), (10, 6), (10,)))
    ups = torch.randn(4, 9, 5, generator=g)
    y = gated._GatedStage.apply(x, w, b, None, None, "sigmoid")
    v, s = torch.nn.functional.linear(x, w, b).chunk(2, -1)
    z = v * torch.sigmoid(s)
    for many in (lambda out: torch.autograd.grad(out, (x, w, b), ups, is_grads_batched=True, retain_graph=True),
                 lambda out: torch.func.vmap(lambda u: torch.autograd.grad(out, (x, w, b), u, retain_graph=True))(ups)):
        for a, r in zip(many(y), many(z)):
            assert torch.equal(a, r) and not a.requires_grad
    assert [name for name, _ in calls] == ["ews_gated_forward"]
