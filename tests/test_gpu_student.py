"""The operators inside a token model's blocks together: a recurrent student (lookup, gated recurrence, gated channel stage)
trained from a teacher's top logits, in training, decoding and captured graphs, and how each stands with torch's other ways
to differentiate. Against the same model in float64 in torch operations.

The whole model's gradients go through two layers, so they are compared as vectors: a float32 model is off by some hundreds
of roundings of 2^-24 of its vectors' lengths (the products' sums of up to 96 numbers, the recurrence's 40 steps, the
loss): 2^-24 times 500 is 3e-5. A bfloat16 model rounds every layer's result once, seven of them from the tokens to the
loss and again on the way back, each by 2^-9 of the vector's length at most on average: 14 of them, added, are 0.027."""

import pytest
import torch
from torch.autograd import forward_ad

import ews_mi355x as E

pytestmark = pytest.mark.gpu

DEV = "cuda"
V, H, F, K = 203, 48, 96, 7
BAR = {torch.float32: 3e-5, torch.bfloat16: 0.027}


def _params(dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def t(*shape, scale):
        return (scale * torch.randn(*shape, generator=g, device=DEV)).to(dtype).requires_grad_()

    return dict(table=t(V, H, scale=1.0), mix=t(2 * H, H, scale=H**-0.5), up=t(2 * F, H, scale=H**-0.5),
                up_bias=t(2 * F, scale=0.2), down=t(H, F, scale=F**-0.5), head=t(V, H, scale=H**-0.5),
                head_bias=t(V, scale=0.2))


def _data(B, L, seed=0):
    g = torch.Generator(device=DEV).manual_seed(100 + seed)
    tokens = torch.randint(0, V, (B, L), generator=g, device=DEV)
    mask = torch.arange(L, device=DEV)[None] < torch.randint(L // 2, L + 1, (B, 1), generator=g, device=DEV)
    index = torch.rand(B, L, V, generator=g, device=DEV).argsort(-1)[..., :K].clone()
    index[torch.rand(B, L, K, generator=g, device=DEV) < 0.1] = -1
    return tokens, mask, index, 2.0 * torch.randn(B, L, K, generator=g, device=DEV)


def _rows(p, tokens, mask=None, state=None, last=None):
    x = E.embedding_lookup(tokens, p["table"], scale=0.5)
    value, gate = torch.nn.functional.linear(x, p["mix"]).chunk(2, -1)
    h, last = E.gated_scan(value, gate, state=state, mask=mask, last=last)
    x = x + h
    y = E.gated_linear(x, p["up"], p["up_bias"], activation="silu")
    return x + torch.nn.functional.linear(y, p["down"]), last


def _loss(p, tokens, mask, index, logits, reduction="mean"):
    rows, last = _rows(p, tokens, mask)
    index = index.masked_fill(~mask[..., None], -1)
    loss = E.linear_distillation(rows, p["head"], index, logits, bias=p["head_bias"], temperature=2.0,
                                 reduction=reduction)
    return loss, rows, last


def _loss64(p, tokens, mask, index, logits):
    p = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    x = 0.5 * p["table"][tokens]
    value, gate = (x @ p["mix"].t()).chunk(2, -1)
    a, s, hs = torch.sigmoid(gate), torch.zeros_like(x[:, 0]), []
    for t in range(tokens.shape[1]):
        on = mask[:, t, None]
        s = torch.where(on, a[:, t] * s + (1 - a[:, t]) * value[:, t], s)
        hs.append(s)
    x = x + torch.stack(hs, 1)
    v, g = (x @ p["up"].t() + p["up_bias"]).chunk(2, -1)
    rows = x + (v * g * torch.sigmoid(g)) @ p["down"].t()
    z = (rows @ p["head"].t() + p["head_bias"]) / 2.0
    has = (index >= 0) & mask[..., None]
    kept = has.any(-1)
    t = torch.where(kept[..., None], (logits.double() / 2.0).masked_fill(~has, -float("inf")), 0.0)
    logp = torch.log_softmax(t, -1)
    each = torch.where(has, logp.exp() * (logp.masked_fill(~has, 0.0)
                                          - torch.log_softmax(z, -1).gather(-1, index.clamp(min=0))), 0.0)
    loss = 4.0 * torch.where(kept, each.sum(-1), 0.0).sum() / kept.sum().clamp(min=1)  # of no rows: 0
    return loss, p, s


def _near(a, r, bar, what):
    off = float((a.double() - r).norm() / r.norm().clamp(min=1e-30))
    assert off <= bar, (what, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L", [(3, 40), (1, 1), (5, 1), (2, 700)])
def test_training_step(B, L, dtype):
    p, data = _params(dtype), _data(B, L)
    loss, _, last = _loss(p, *data)
    want, p64, s = _loss64(p, *data)
    _near(loss.detach(), want.detach(), BAR[dtype], "loss")
    _near(last.detach(), s.detach(), BAR[dtype], "last state")
    got = torch.autograd.grad(loss, list(p.values()))
    exact = torch.autograd.grad(want, list(p64.values()))
    for name, a, r in zip(p, got, exact):
        _near(a, r, BAR[dtype], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decoding_follows_the_whole_sequence(dtype):
    """A prompt, then a token at a time with the state in place, eagerly and in a captured graph replayed for every token:
    the graph gives the eager bits, and both the rows of the whole sequence but for roundings."""
    p, (tokens, _, _, _) = _params(dtype), _data(2, 30)
    with torch.no_grad():
        whole, _ = _rows(p, tokens)
        state = torch.empty(2, H, device=DEV)
        rows = [_rows(p, tokens[:, :9], last=state)[0]]
        start = state.clone()
        for t in range(9, 30):
            rows.append(_rows(p, tokens[:, t:t + 1], state=state, last=state)[0])
        eager = torch.cat(rows, 1)
        _near(eager, whole.double(), BAR[dtype], "rows")
        held, now = start.clone(), tokens[:, 9:10].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _rows(p, now, state=held.clone(), last=torch.empty_like(held))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = _rows(p, now, state=held, last=held)
        held.copy_(start)
        for t in range(9, 30):
            now.copy_(tokens[:, t:t + 1])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[:, 0], eager[:, t])
        assert torch.equal(held, state)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,B,L", [(torch.float32, 3, 40), (torch.bfloat16, 2, 700)])
def test_replayed_steps_match_eager_ones(dtype, B, L, reduction):
    p, data = _params(dtype), _data(B, L)

    def step():
        loss, rows, last = _loss(p, *data, reduction=reduction)
        up = torch.ones_like(loss) if reduction == "none" else None
        return [loss.detach(), rows.detach(), last.detach(), *torch.autograd.grad(loss, list(p.values()), up)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        first = step()
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):  # two graphs of one pool, replayed in turn
        second = step()
    for n in range(4):
        for t, new in zip(data, _data(B, L, seed=1 + n)):
            t.copy_(new)
        graphs[n % 2].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (first, second)[n % 2]]
        want = step()
        torch.cuda.synchronize()
        for a, r in zip(got, want):
            assert torch.equal(a, r)


def test_two_streams_at_once():
    """The same calls on two streams at a time give the bits that they give alone."""
    p = _params(torch.bfloat16)
    datas = [_data(2, 700, seed=s) for s in range(2)]

    def step(data):
        loss, _, _ = _loss(p, *data)
        return [loss.detach(), *torch.autograd.grad(loss, list(p.values()))]

    want = [step(d) for d in datas]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in datas]
    for _ in range(3):
        got = []
        for s, d in zip(streams, datas):
            with torch.cuda.stream(s):
                got.append(step(d))
        torch.cuda.synchronize()
        for a, r in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, r))


def _calls(dual):
    x, w, b = torch.randn(3, 8, device=DEV), torch.randn(10, 8, device=DEV), torch.randn(10, device=DEV)
    seq, index = torch.randn(2, 4, 8, device=DEV), torch.tensor([[1, 2]] * 3, device=DEV)
    state, logits = torch.randn(2, 8, device=DEV), torch.randn(3, 2, device=DEV)
    yield "gated, x", lambda: E.gated_linear(dual(x), w, b)
    yield "gated, weight", lambda: E.gated_linear(x, dual(w), b)
    yield "gated, bias", lambda: E.gated_linear(x, w, dual(b))
    yield "gated, gate", lambda: E.gated_linear(x, w, b, dual(w), b)
    yield "scan, x", lambda: E.gated_scan(dual(seq), seq)
    yield "scan, gate", lambda: E.gated_scan(seq, dual(seq))
    yield "scan, state", lambda: E.gated_scan(seq, seq, state=dual(state))
    yield "distillation, hidden", lambda: E.linear_distillation(dual(x), w, index, logits)
    yield "distillation, weight", lambda: E.linear_distillation(x, dual(w), index, logits, reduction="none")
    yield "distillation, logits", lambda: E.linear_distillation(x, w, index, dual(logits))


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(no_grad):
    with forward_ad.dual_level():
        for name, call in _calls(lambda x: forward_ad.make_dual(x, torch.ones_like(x))):
            print(name, flush=True)
            with torch.set_grad_enabled(not no_grad), pytest.raises(NotImplementedError):
                call()
        for _, call in _calls(lambda x: x):
            call()


def test_a_last_state_that_is_given():
    """What is written is seen by graphs that saved it; what overlaps is refused; nothing is recorded."""
    x, gate = torch.randn(2, 5, 8, device=DEV), torch.randn(2, 5, 8, device=DEV)
    last = torch.zeros(2, 8, device=DEV)
    w = torch.ones(2, 8, device=DEV, requires_grad=True)
    y, before = (w * last).sum(), last._version
    E.gated_scan(x, gate, last=last)
    assert last._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    flat = torch.zeros(40, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        E.gated_scan(x, gate, state=flat[:16].view(2, 8), last=flat[8:24].view(2, 8))
    E.gated_scan(x, gate, state=flat[:16].view(2, 8), last=flat[16:32].view(2, 8))
    with pytest.raises(ValueError, match="overlaps"):
        E.gated_scan(x, gate, last=x.view(-1)[:16].view(2, 8))
    with pytest.raises(ValueError, match="contiguous"):
        E.gated_scan(x, gate, last=torch.zeros(8, 2, device=DEV).t())
    with pytest.raises(ValueError, match="no_grad"):
        E.gated_scan(x.requires_grad_(), gate, last=last)
    with torch.inference_mode():
        s = torch.zeros(2, 8, device=DEV)
        h, out = E.gated_scan(torch.randn(2, 5, 8, device=DEV), gate, state=s, last=s)
        assert out is s and bool(s.any())


@pytest.mark.parametrize("stage", ["glu", "gelu_glu"])
def test_the_blocks_channel_stage(stage):
    """Fused or by its maps: the same but for float32's rounding; maps that are more than maps are called."""
    block = E.EWSBlock(40, m=6, n=2, a_param=E.AParamEFM(torch.randn(6)), leaf="series", series_q=6, channel_stage=stage,
                       dropout_rate=0.0, key=3).to(DEV)
    x = torch.randn(2, 30, 40, device=DEV)

    def grads(fused):
        block.fused_channel = fused
        y = block(x)
        return [y.detach(), *torch.autograd.grad(y.square().sum(), list(block.parameters()), allow_unused=True)]

    for a, r in zip(grads(True), grads(False)):
        if r is not None:
            # a stage's sums of 40 numbers, and the parameters' of 60 rows: some hundreds of roundings
            assert float((a - r).norm() / r.norm().clamp(min=1e-20)) <= 3e-5
    block.fused_channel = True
    calls = []
    handle = block.ff1.register_forward_hook(lambda m, i, out: calls.append(1) or out * 0.5)
    half = block(x)
    handle.remove()
    assert calls and not torch.equal(half, block(x))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        block._channel(x)  # torch's own maps decide what autocast does
    calls.clear()
    block.ff1.register_forward_pre_hook(lambda m, i: calls.append(1))
    block(x)
    assert calls
