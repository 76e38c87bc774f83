"""What ``gated_scan`` refuses, before any device is touched, and the library's own checks."""

import ctypes

import pytest
import torch

import ews_mi355x as E
from ews_mi355x import _native as nat


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kwargs,error,says", [
    (dict(form="log"), ValueError, "form must be one of"),
    (dict(x=_x(4, 5)), ValueError, r"x must be \(B, L, D\)"),
    (dict(x=_x(2, 4, 0), gate=_x(2, 4, 0)), ValueError, "D >= 1"),
    (dict(gate=_x(2, 4, 6)), ValueError, "gate must be"),
    (dict(), RuntimeError, "HIP device"),
])
def test_refusals(kwargs, error, says):
    args = dict(x=_x(2, 4, 5), gate=_x(2, 4, 5), **{k: v for k, v in kwargs.items() if k not in ("x", "gate")})
    args.update({k: v for k, v in kwargs.items() if k in ("x", "gate")})
    with pytest.raises(error, match=says):
        E.gated_scan(**args)


def _desc(**kw):
    base = dict(x_batch=40, x_step=8, gate_batch=40, gate_step=8, mask_batch=5, batch=2, length=5, dim=8, dtype=0, form=0)
    base.update(kw)
    return nat.GatedScanDesc(**base)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(form=2), dict(form=-1), dict(batch=0), dict(length=0), dict(dim=0),
                                 dict(dim=(1 << 20) + 1), dict(length=(1 << 28) + 1), dict(x_step=-1),
                                 dict(gate_batch=-8)])
def test_library_refuses(bad):
    lib = nat.load()
    one = ctypes.c_void_p(16)
    d = _desc(**bad)
    assert lib.ews_gated_scan_residual_bytes(d) == 0
    assert lib.ews_gated_scan_forward(d, one, one, None, None, one, one, None, one, None) in (-2, -4)
    assert lib.ews_gated_scan_backward(d, one, one, None, one, None, None, one, one, None, one, None) in (-2, -4)


def test_library_refuses_null():
    lib = nat.load()
    one = ctypes.c_void_p(16)
    d = _desc()
    assert lib.ews_gated_scan_forward(None, one, one, None, None, one, one, None, one, None) == -1
    for hole in range(4):
        p = [one] * 4
        p[hole] = None
        assert lib.ews_gated_scan_forward(d, p[0], p[1], None, None, p[2], p[3], None, None, None) == -1
    long = _desc(length=100000, batch=1)
    assert lib.ews_gated_scan_workspace_bytes(long) > 0
    assert lib.ews_gated_scan_forward(long, one, one, None, None, one, one, None, None, None) == -1
    assert lib.ews_gated_scan_backward(d, one, one, None, None, None, None, one, one, None, None, None) == -1


def test_scratch_is_small():
    lib = nat.load()
    for B, L, D in ((1, 131071, 1024), (8, 4095, 2048), (1, 1 << 20, 8), (4096, 100, 4096)):
        d = _desc(batch=B, length=L, dim=D, x_batch=L * D, x_step=D, gate_batch=L * D, gate_step=D)
        assert lib.ews_gated_scan_residual_bytes(d) <= B * (L // 8 + 1) * D * 4
        assert lib.ews_gated_scan_workspace_bytes(d) <= 4 * B * D * 4 + 4 * (1 << 20)
