"""What ``gated_linear`` refuses before any device is touched, the library's own checks, and its choice of tiles."""

import ctypes

import pytest
import torch

import ews_mi355x as E
from ews_mi355x import _native as nat
from gated_shapes import SHARED, TILES


@pytest.mark.parametrize("change,error,says", [
    (dict(activation="tanh"), ValueError, "activation must be"),
    (dict(weight=torch.zeros(7, 4)), ValueError, r"weight must be \(2 F, H\)"),
    (dict(weight=torch.zeros(8)), ValueError, "weight must be"),
    (dict(weight=torch.zeros(0, 4)), ValueError, "weight must be"),
    (dict(x=torch.zeros(6, 5)), ValueError, "x must be"),
    (dict(bias=torch.zeros(4)), ValueError, "bias must be"),
    (dict(gate_weight=torch.zeros(4, 4)), ValueError, "gate_weight must be"),
    (dict(gate_bias=torch.zeros(4)), ValueError, "goes with gate_weight"),
    (dict(gate_weight=torch.zeros(8, 4), gate_bias=torch.zeros(4)), ValueError, "gate_bias must be"),
    (dict(), RuntimeError, "HIP device"),
])
def test_refusals(change, error, says):
    with pytest.raises(error, match=says):
        E.gated_linear(**{**dict(x=torch.zeros(6, 4), weight=torch.zeros(8, 4)), **change})


def _desc(**kw):
    base = dict(x_stride=4, weight_stride=4, gate_stride=4, rows=6, width=4, features=4, dtype=0, activation=0)
    base.update(kw)
    return nat.GatedDesc(**base)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(activation=4), dict(activation=-1), dict(rows=0), dict(width=0),
                                 dict(features=0), dict(rows=(1 << 24) + 1), dict(x_stride=3), dict(gate_stride=3),
                                 dict(width=1 << 16, x_stride=1 << 16, weight_stride=1 << 16, gate_stride=1 << 16,
                                      features=1 << 20)])
def test_library_refuses(bad):
    lib, one = nat.load(), ctypes.c_void_p(16)
    d = _desc(**bad)
    assert lib.ews_gated_kept_bytes(d) == 0 and lib.ews_gated_workspace_bytes(d, one, one, one, 2) == 0
    assert lib.ews_gated_forward(d, one, one, None, one, None, one, None, one, None) in (-2, -4)
    assert lib.ews_gated_backward(d, one, one, None, one, None, one, one, one, one, None, one, None, one, None) in (-2, -4)


def test_library_refuses_null():
    lib, one, d = nat.load(), ctypes.c_void_p(16), _desc(rows=100, features=100)
    assert lib.ews_gated_forward(None, one, one, None, one, None, one, None, one, None) == -1
    for hole in range(5):
        p = [one] * 5
        p[hole] = None
        assert lib.ews_gated_forward(d, p[0], p[1], None, p[2], None, p[3], None, p[4], None) == -1
    for hole in range(6):
        p = [one] * 6
        p[hole] = None
        assert lib.ews_gated_backward(d, p[0], p[1], None, p[2], None, p[3], p[4], one, one, None, one, None, p[5],
                                      None) == -1


@pytest.mark.parametrize("case", list(TILES))
def test_tiles(case):
    name, N, H, F = case
    d = _desc(rows=N, width=H, features=F, x_stride=H, weight_stride=H, gate_stride=H,
              dtype=nat.DTYPE_F32 if name == "float32" else nat.DTYPE_BF16)
    tile = (ctypes.c_int32 * 5)()
    for product, want in enumerate(TILES[case]):
        assert nat.load().ews_gated_tile(d, product, tile) == 0
        assert tuple(tile[:2]) == want, product


@pytest.mark.parametrize("dtype", [nat.DTYPE_F32, nat.DTYPE_BF16])
@pytest.mark.parametrize("size", list(SHARED))
def test_shared_tiles(size, dtype):
    N, H, F = size
    d = _desc(rows=N, width=H, features=F, x_stride=H, weight_stride=H, gate_stride=H, dtype=dtype)
    tile = (ctypes.c_int32 * 5)()
    product, alone, tiles = SHARED[size]
    assert nat.load().ews_gated_tile(d, product, tile) == 0
    assert tuple(tile) == (256, 256, 1, alone, tiles)


def test_scratch_of_what_is_read_where_it_is():
    """bfloat16 rows at multiples of 16 bytes and of whole k blocks need no copies; few rows never do."""
    lib = nat.load()
    d = _desc(rows=4096, width=128, features=512, x_stride=128, weight_stride=128, gate_stride=128, dtype=1)
    assert lib.ews_gated_workspace_bytes(d, 4096, 1 << 20, 1 << 21, nat.GATED_KEEP) == 0
    assert lib.ews_gated_workspace_bytes(d, 4098, 1 << 20, 1 << 21, nat.GATED_KEEP) == 4096 * 128 * 2
    assert lib.ews_gated_workspace_bytes(d, 4096, 1 << 20, (1 << 21) + 2, nat.GATED_KEEP) == 2 * 512 * 128 * 2
    few = _desc(rows=64, width=130, features=512, x_stride=130, weight_stride=130, gate_stride=130)
    assert lib.ews_gated_workspace_bytes(few, 4098, 6, 10, nat.GATED_FORWARD) == 0
    assert lib.ews_gated_workspace_bytes(few, 4098, 6, 10, nat.GATED_KEEP) == 0
    some = _desc(rows=33, width=130, features=512, x_stride=130, weight_stride=130, gate_stride=130, dtype=1)
    assert lib.ews_gated_workspace_bytes(some, 4098, 6, 10, nat.GATED_FORWARD) > 0


@pytest.mark.parametrize("N,H,F", [
    (1 << 24, 4, 4), ((1 << 24) + 1, 4, 4), (6, 1 << 16, 100), (6, (1 << 16) + 1, 100), (6, 100, 1 << 20),
    (6, 100, (1 << 20) + 1), (1 << 24, 512, 4), (1 << 24, 513, 4), (6, 1 << 13, 1 << 20), (6, (1 << 13) + 1, 1 << 20),
    (1 << 24, 4, 1024), (1 << 24, 4, 1025), ((1 << 23) - 1, 1024, 65), ((1 << 23) + 1, 1024, 65), (1, 1, 1),
])
def test_sizes_that_fit_are_the_librarys(N, H, F):
    from ews_mi355x.gated import _fits

    tile = (ctypes.c_int32 * 5)()
    d = _desc(rows=N, width=H, features=F, x_stride=H, weight_stride=H, gate_stride=H)
    assert (nat.load().ews_gated_tile(d, 0, tile) == 0) == _fits(N, H, F)


def test_sizes_that_do_not_fit_are_refused():
    x = torch.zeros(1, 4).expand((1 << 24) + 1, 4)
    with pytest.raises(ValueError, match="rows"):
        E.gated_linear(x, torch.zeros(8, 4))


def test_narrow_maps_keep_nothing():
    lib = nat.load()
    for H, F, narrow in ((64, 64, True), (1, 1, True), (65, 64, False), (64, 65, False)):
        d = _desc(rows=1 << 20, width=H, features=F, x_stride=H, weight_stride=H, gate_stride=H)
        assert (lib.ews_gated_kept_bytes(d) == 0) == narrow
        if narrow:
            assert lib.ews_gated_workspace_bytes(d, 4098, 6, 10, nat.GATED_KEEP) == 0
            assert 0 < lib.ews_gated_workspace_bytes(d, 4098, 6, 10, nat.GATED_BACKWARD) <= 512 * 128 * 65 * 4
