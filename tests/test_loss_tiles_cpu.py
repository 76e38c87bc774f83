"""The rule that chooses linear cross entropy's tiles, at the sizes that the device tests run: a change of the rule that
moves one of them to another tile fails here, so that no tile can fall out of the tests unseen."""

import ctypes

import pytest

from ews_mi355x import _native as nat
from loss_shapes import FEW32, FLAT, LARGE, MEDIUM, MORE32, TILES

ALIGNED = ctypes.c_void_p(4096)


def _tile(key, product, train=1, weight=ALIGNED, **kw):
    dtype, N, H, V, reduction = key
    base = dict(hidden_stride=H, weight_stride=H, ignore_index=-100, rows=N, hidden=H, vocab=V,
                dtype=0 if dtype == "float32" else 1, bias_dtype=0, reduction=nat.LOSS_REDUCTIONS[reduction])
    out = (ctypes.c_int32 * 4)()
    code = nat.load().ews_loss_tile(nat.LossDesc(**{**base, **kw}), weight, train, product, out)
    return code if code else tuple(out)


@pytest.mark.parametrize("key", TILES, ids=str)
def test_tiles(key):
    assert tuple(_tile(key, q)[:2] for q in range(3)) == TILES[key]
    assert _tile(key, 0, train=0)[:2] == TILES[key][0]


def test_every_tile_of_every_product_is_run():
    """What the kernels are built for."""
    rows = {LARGE, MEDIUM, FLAT, FEW32, MORE32}
    for dtype, logits, hidden, weight in (("float32", rows, rows, {LARGE, MEDIUM}),
                                          ("bfloat16", {LARGE, MEDIUM, FLAT}, {LARGE, MEDIUM, FLAT}, {LARGE, MEDIUM})):
        mine = [tiles for key, tiles in TILES.items() if key[0] == dtype]
        for q, want in enumerate((logits, hidden, weight)):
            assert want <= {tiles[q] for tiles in mine}


def test_refusals():
    key = next(iter(TILES))
    assert _tile(key, 3) == -4 and _tile(key, -1) == -4 and _tile(key, 1, train=0) == -4
    assert _tile(key, 0, rows=0) == -2
    assert nat.load().ews_loss_tile(None, ALIGNED, 1, 0, (ctypes.c_int32 * 4)()) == -1
