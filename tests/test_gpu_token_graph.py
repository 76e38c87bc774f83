"""A token model's ends captured as a HIP graph: lookup, loss, gradients and clipping, replayed on new data with the
same calls made eagerly between the replays. Every sum has a fixed order, so a replay gives the eager bits."""

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _step(tokens, targets, table, head, bias, reduction):
    x = E.embedding_lookup(tokens, table, scale=3.0, padding_idx=0)
    loss = E.linear_cross_entropy(x, head, targets, bias=bias, reduction=reduction)
    up = torch.ones_like(loss) if reduction == "none" else None
    grads = torch.autograd.grad(loss, [table, head, bias], up)
    norm, clipped = E.clip_grads(grads, 0.05)
    return [loss.detach(), norm, *clipped]


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,n,H,V", [(torch.float32, 40, 72, 301), (torch.bfloat16, 700, 192, 2111)])
def test_replays_match_eager(dtype, n, H, V, reduction):
    g = torch.Generator(device=DEV).manual_seed(n)

    def data():
        tokens = torch.randint(V, (n,), generator=g, device=DEV)
        targets = torch.randint(V, (n,), generator=g, device=DEV)
        targets[torch.rand(n, generator=g, device=DEV) < 0.2] = -100
        return tokens, targets

    table, head, bias = ((torch.randn(s, generator=g, device=DEV) * 0.3).to(dtype).requires_grad_()
                         for s in ((V, H), (V, H), (V,)))
    tokens, targets = data()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on a side stream, as graph capture asks
        _step(tokens, targets, table, head, bias, reduction)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(tokens, targets, table, head, bias, reduction)
    for _ in range(4):
        for t, new in zip((tokens, targets), data()):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(tokens, targets, table, head, bias, reduction)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
