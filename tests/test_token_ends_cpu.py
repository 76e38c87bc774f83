"""CPU checks of the operators around a token model's blocks (ews_embed.hip, ews_loss.hip, ews_clip.hip): the host
layer's refusals, and the C ABI's error codes and scratch sizes (no launch: there is no GPU here)."""

import ctypes

import pytest
import torch

import ews_mi355x as E
from ews_mi355x import _native as nat

NULL = ctypes.c_void_p(0)


def test_host_layer_refuses_cpu_tensors_and_bad_shapes():
    w, t = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP device only"):
        E.embedding_lookup(t, w)
    with pytest.raises(RuntimeError, match="HIP device only"):
        E.linear_cross_entropy(torch.zeros(3, 8), w, t)
    with pytest.raises(RuntimeError, match="HIP device only"):
        E.clip_grads([w], 1.0)
    with pytest.raises(ValueError, match="weight must be"):
        E.embedding_lookup(t, w[0])
    with pytest.raises(ValueError, match="hidden must be"):
        E.linear_cross_entropy(torch.zeros(3, 7), w, t)
    with pytest.raises(ValueError, match="targets must be"):
        E.linear_cross_entropy(torch.zeros(3, 8), w, t[:2])
    with pytest.raises(ValueError, match="bias must be"):
        E.linear_cross_entropy(torch.zeros(3, 8), w, t, bias=torch.zeros(4))
    with pytest.raises(ValueError, match="reduction must be"):
        E.linear_cross_entropy(torch.zeros(3, 8), w, t, reduction="max")
    with pytest.raises(ValueError, match="max_norm"):
        E.clip_grad_norm_([], -1.0)


def _embed(**kw):
    base = dict(count=10, weight_stride=16, padding=-1, width=16, vocab=9, dtype=0, token_bytes=8, scale=1.0)
    return nat.EmbedDesc(**{**base, **kw})


def test_embed_error_codes():
    lib = nat.load()
    assert lib.ews_embed_forward(_embed(), NULL, NULL, NULL, NULL) == -1
    assert lib.ews_embed_workspace_bytes(_embed(count=1000)) > 0
    assert lib.ews_embed_workspace_bytes(_embed(count=256)) == 0
    for bad, code in ((dict(count=0), -2), (dict(count=2**25 + 1), -2), (dict(width=0), -2), (dict(vocab=0), -2),
                      (dict(weight_stride=15), -2), (dict(vocab=2**25 + 1), -2), (dict(dtype=2), -4),
                      (dict(token_bytes=2), -4)):
        assert lib.ews_embed_forward(_embed(**bad), NULL, NULL, NULL, NULL) == code, bad
        assert lib.ews_embed_backward(_embed(**bad), NULL, NULL, NULL, NULL, NULL) == code, bad
        assert lib.ews_embed_workspace_bytes(_embed(**bad)) == 0, bad


def _loss(**kw):
    base = dict(hidden_stride=64, weight_stride=64, ignore_index=-100, rows=10, hidden=64, vocab=100, dtype=0,
                bias_dtype=0, reduction=1)
    return nat.LossDesc(**{**base, **kw})


def test_loss_error_codes():
    lib = nat.load()
    nulls = [NULL] * 7
    assert lib.ews_loss_forward(_loss(), *nulls) == -1
    assert lib.ews_loss_train(_loss(), *nulls, *[NULL] * 4) == -1
    for bad, code in ((dict(rows=0), -2), (dict(hidden=0), -2), (dict(vocab=0), -2), (dict(hidden_stride=63), -2),
                      (dict(weight_stride=63), -2), (dict(vocab=2**22 + 1), -2), (dict(rows=2**22 + 1), -2),
                      (dict(hidden=2**16 + 1, hidden_stride=2**17, weight_stride=2**17), -2), (dict(dtype=3), -4),
                      (dict(bias_dtype=-1), -4), (dict(reduction=3), -4)):
        assert lib.ews_loss_forward(_loss(**bad), *nulls) == code, bad
        assert lib.ews_loss_train(_loss(**bad), *nulls, *[NULL] * 4) == code, bad
        assert lib.ews_loss_workspace_bytes(_loss(**bad), 1) == 0, bad


def test_loss_scratch_does_not_grow_with_the_logits():
    lib = nat.load()

    def scratch(rows, train):
        return lib.ews_loss_workspace_bytes(
            _loss(rows=rows, hidden=512, hidden_stride=512, weight_stride=512, vocab=100003, dtype=1), train)

    inputs = (65536 * 2 + 100003 * 3) * 512 * 2 + 100003 * 512 * 4  # packed rows and weights, the gradient's sums
    assert scratch(65536, 1) < (2 << 30) * 1.1 + inputs < 65536 * 100003 * 2
    assert scratch(65536, 0) < inputs + (1 << 30)


def test_clip_error_codes():
    lib = nat.load()
    one = (ctypes.c_uint64 * 1)(4096)
    count, dtype = (ctypes.c_int64 * 1)(8), (ctypes.c_int32 * 1)(0)
    assert lib.ews_clip_workspace_bytes(1, count) == 8
    assert lib.ews_clip(1, one, one, count, dtype, 1.0, 1, NULL, NULL, NULL) == -1
    assert lib.ews_clip(1, NULL, one, count, dtype, 1.0, 1, NULL, NULL, NULL) == -1
    assert lib.ews_clip(-1, one, one, count, dtype, 1.0, 1, NULL, NULL, NULL) == -2
    assert lib.ews_clip(1, one, one, (ctypes.c_int64 * 1)(-1), dtype, 1.0, 1, NULL, NULL, NULL) == -2
    assert lib.ews_clip(1, one, one, count, (ctypes.c_int32 * 1)(5), 1.0, 1, NULL, NULL, NULL) == -4
    assert lib.ews_loss_scale(_loss(), NULL, NULL, NULL, NULL, NULL) == -1
    assert lib.ews_loss_scale(_loss(rows=0), NULL, NULL, NULL, one, NULL) == -2
