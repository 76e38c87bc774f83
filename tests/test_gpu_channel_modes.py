"""Gated channel stages of a block in the modes of differentiation that torch's operations have: what ``gated_linear``
does not do, the stage's maps do."""

import pytest
import torch
from torch.autograd import forward_ad

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _block(stage):
    return E.EWSBlock(40, m=6, n=2, a_param=E.AParamEFM(torch.randn(6)), leaf="series", series_q=6, channel_stage=stage,
                      dropout_rate=0.0, key=3).to(DEV)


@pytest.mark.parametrize("stage", ["glu", "gelu_glu"])
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode(stage, no_grad):
    """A tangent of a map's weight or bias, and of what goes in, takes the maps; none of them does not."""
    block = _block(stage)
    x = torch.randn(2, 30, 40, device=DEV)
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        plain = block._channel(x)
        block.fused_channel = False
        want = block._channel(x)
        block.fused_channel = True
        assert forward_ad.unpack_dual(plain).tangent is None
        for name in ("weight", "bias", "x"):
            outs = []
            for fused in (True, False):
                block.fused_channel = fused
                if name == "x":
                    outs.append(block._channel(forward_ad.make_dual(x, torch.ones_like(x))))
                    continue
                p = getattr(block.ff1, name)
                delattr(block.ff1, name)
                setattr(block.ff1, name, forward_ad.make_dual(p.detach(), torch.ones_like(p)))
                outs.append(block._channel(x))
                delattr(block.ff1, name)
                setattr(block.ff1, name, p)
            a, b = (forward_ad.unpack_dual(o) for o in outs)
            assert torch.equal(a.primal, want) and torch.equal(a.tangent, b.tangent) and bool(a.tangent.any())
        block.fused_channel = True


@pytest.mark.parametrize("stage", ["glu", "gelu_glu"])
def test_second_derivatives(stage):
    """Of a stage's weights, through a block: those of the maps."""
    block = _block(stage)
    x = torch.randn(2, 30, 40, device=DEV)
    weights = [block.ff1.weight, block.ff1.bias]
    got = []
    for fused in (True, False):
        block.fused_channel = fused
        grads = torch.autograd.grad(block(x).square().sum(), weights, create_graph=True)
        got.append([*grads, *torch.autograd.grad(sum(g.square().sum() for g in grads), weights)])
    for a, r in zip(*got):
        # sums of 40 numbers and of 60 rows, twice: some hundreds of float32 roundings
        assert float((a - r).detach().norm() / r.detach().norm()) <= 3e-5
