"""The memory that linear cross entropy takes on the device."""

import pytest
import torch

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scoring_a_few_rows_does_not_copy_the_weight(dtype):
    V, H = 50000, 1024
    w = torch.randn(V, H, device=DEV).to(dtype)
    h, t = torch.randn(3, H, device=DEV).to(dtype), torch.tensor([1, 2, 3], device=DEV)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with torch.no_grad():
        E.linear_cross_entropy(h, w, t, reduction="none")
    assert torch.cuda.max_memory_allocated() - before < 4 << 20


SCRATCH = [(141, 396, 1980), (256, 64, 1000), (200, 1000, 333), (33, 257, 4001), (7, 4096, 700), (300, 130, 900),
           (600, 128, 9000), (700, 70, 7001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,H,V", SCRATCH)
def test_scratch_of_a_weight_holds_what_its_call_writes(N, H, V, dtype, monkeypatch):
    """Beyond the bytes that the library asks for with the weight's address a workspace stays as it was."""
    from ews_mi355x import loss as module

    spaces = []

    def workspace(self, train):
        size = module.nat.load().ews_loss_workspace_bytes_for(self.desc, self.weight.data_ptr(), train)
        whole = torch.full((size + (64 << 20),), 91, dtype=torch.uint8, device=DEV)
        spaces.append((whole, size))
        return whole[:size]

    monkeypatch.setattr(module._Call, "workspace", workspace)
    g = torch.Generator(device=DEV).manual_seed(N)
    w = torch.randn(V, H, generator=g, device=DEV).to(dtype)
    h = torch.randn(N, H, generator=g, device=DEV).to(dtype)
    b = torch.randn(V, generator=g, device=DEV)
    t = torch.randint(0, V, (N,), generator=g, device=DEV)
    odd = torch.empty(V * H + 1, device=DEV, dtype=dtype)[1:].view(V, H)
    results = []
    for weight in (w, odd.copy_(w)):
        weight = weight.detach().requires_grad_()
        for reduction in ("none", "mean"):
            hidden = h.detach().requires_grad_()
            rows = E.linear_cross_entropy(hidden, weight, t, bias=b, reduction=reduction)
            results.append((rows.detach(), *torch.autograd.grad(rows, [hidden, weight], torch.ones_like(rows))))
        with torch.no_grad():
            E.linear_cross_entropy(h, weight, t, bias=b)
    torch.cuda.synchronize()
    assert len(spaces) == 6
    for whole, size in spaces:
        assert bool((whole[size:] == 91).all())
    for one, other in zip(results[:2], results[2:]):  # however W is read, its numbers are the same
        for a, c in zip(one, other):
            assert torch.allclose(a.float(), c.float(), rtol=0.0, atol=2.0**-7 * float(a.float().abs().max()))
