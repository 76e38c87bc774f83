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
