"""Limits and scratch of the token model's ends as the C ABI answers them (no launch: there is no GPU here)."""

import ctypes

import pytest

from ews_mi355x import _native as nat

NULL = ctypes.c_void_p(0)


def _embed(**kw):
    base = dict(count=1000, weight_stride=16, padding=-1, width=16, vocab=9, dtype=0, token_bytes=8, scale=1.0)
    return nat.EmbedDesc(**{**base, **kw})


@pytest.mark.parametrize("count", [200, 1000])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("vocab,width,taken", [(2**25, 65, True), (2**22, 4096, True), (2**25, 4096, True),
                                               (2**25, 2**20, False), (2**20, 2**19, False), (1, 2**20, True)])
def test_lookup_and_gradient_take_the_same_sizes(vocab, width, taken, dtype, count):
    """A size is refused (-2) by the forward, the scratch query and the backward alike, or by none (-1: no tensors)."""
    lib = nat.load()
    d = _embed(count=count, weight_stride=width, width=width, vocab=vocab, dtype=dtype)
    code = -1 if taken else -2
    assert lib.ews_embed_forward(d, NULL, NULL, NULL, NULL) == code
    assert lib.ews_embed_backward(d, NULL, NULL, NULL, NULL, NULL) == code
    assert (lib.ews_embed_workspace_bytes(d) > 0) == (taken and count > 256)


def _scratch(rows, train, hidden=512, vocab=100003, dtype=0, reduction=1):
    d = nat.LossDesc(hidden_stride=hidden, weight_stride=hidden, ignore_index=-100, rows=rows, hidden=hidden,
                     vocab=vocab, dtype=dtype, bias_dtype=0, reduction=reduction)
    return nat.load().ews_loss_workspace_bytes(d, train)


@pytest.mark.parametrize("rows,hidden", [(65536, 64), (1 << 20, 64), (8192, 512), (600, 64), (600, 4096)])
def test_float32_scores_keep_256_mib_of_slabs(rows, hidden):
    """Beside the planes of rows and weight and eight numbers a row or token at most."""
    planes = (rows + 100003) * ((hidden + 63) // 64 * 64) * 6
    assert _scratch(rows, 0, hidden) <= planes + (256 << 20) + 32 * (rows + 100003 + 1024)


@pytest.mark.parametrize("rows,train,most", [(1, 0, 2 << 20), (512, 0, 140 << 20), (64, 1, 180 << 20)])
def test_float32_weight_read_as_it_is_has_no_copy(rows, train, most):
    """Few rows: W (1.6 GB here, its planes 2.5) is not copied. A row has a slab's eight bytes for 32 tokens, in
    training ten bytes a token, and the results of up to 128 splits of dh."""
    splits = 128 * rows * 4096 * 4 if train else 0
    assert _scratch(rows, train, 4096) <= most + splits


@pytest.mark.parametrize("train", [0, 1])
@pytest.mark.parametrize("rows,hidden,dtype", [(1, 4096, 1), (1000, 4096, 1), (1, 4000, 1), (3, 4096, 0),
                                               (7000, 512, 0)])
def test_scratch_of_a_weight_at_an_address(rows, hidden, dtype, train):
    """The query without the address holds any weight's; with it, a bfloat16 weight that is read where it is has no
    copy."""
    lib = nat.load()
    d = nat.LossDesc(hidden_stride=hidden, weight_stride=hidden, ignore_index=-100, rows=rows, hidden=hidden,
                     vocab=100003, dtype=dtype, bias_dtype=0, reduction=0)
    any_weight = lib.ews_loss_workspace_bytes(d, train)
    aligned, odd = (lib.ews_loss_workspace_bytes_for(d, ctypes.c_void_p(a), train) for a in (4096, 4098))
    copy = 100003 * ((hidden + 63) // 64 * 64) * 2
    assert max(aligned, odd) == any_weight
    assert aligned == any_weight - (copy + 255) // 256 * 256 if dtype == 1 and hidden % 64 == 0 else aligned == odd
    if rows == 1 and hidden == 4096 and not train:
        assert aligned < 1 << 20
    assert lib.ews_loss_workspace_bytes_for(None, None, train) == 0
    d.rows = 0
    assert lib.ews_loss_workspace_bytes_for(d, ctypes.c_void_p(4096), train) == 0
