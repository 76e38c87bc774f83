"""What is timed of the operators around the blocks of a token model's training step: the embedding and its gradient,
the head's softmax cross entropy with its gradients, and the clipping of all gradients by their global norm.

Every case runs one whole call on inputs made from the seed. Where ``own`` is false ``run`` computes the operator in
its plain form with elementary torch operations in float32, rounded once at the end; where it is true ``run`` calls
the package. ``exact`` restates the definition in float64.

Kinds of case:

    loss   ``linear_cross_entropy`` of N rows of width H against a vocabulary of V
    embed  ``embedding_lookup`` of n tokens in a (V, H) table
    clip   ``clip_grads`` / ``clip_grad_norm_`` over the gradients of a stack of blocks with an embedding and a head
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "exponentially-weighted-signature_amd")

IGNORE = -100
NORM_EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}

_LOSS = dict(kind="loss", N=1, H=1, V=1, dtype="float32", bias=False, reduction="mean", train=True, ignored=0.1)
_EMBED = dict(kind="embed", n=1, H=1, V=1, dtype="float32", scale=1.0, pads=0.0, train=True)
_CLIP = dict(kind="clip", blocks=1, H=32, V=8, dtype="float32", clipped=True, in_place=False)

LARGEST = 16384 * 4096 * 100003  # N H V of the largest loss
LARGEST_ROWS = 131071 * 2048  # n H of the largest embedding
LARGEST_TABLE = 100003 * 2048  # V H of its table
LARGEST_GRADS = 3_100_000_000  # numbers in the largest set of gradients


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # A small stack on a short batch: launches and their latency are most of the step's end.
        dict(_LOSS, name="loss_small_f32_train", N=256, H=64, V=1000, bias=True),
        # A float32 model of the package's default type with a head's bias, odd row count.
        dict(_LOSS, name="loss_f32_train", N=4095, H=512, V=32000, bias=True),
        # A bfloat16 training step of ordinary size.
        dict(_LOSS, name="loss_bf16_train", N=8192, H=2048, V=32000, dtype="bfloat16"),
        # The largest: a wide model, a vocabulary of 100k that no tile divides.
        dict(_LOSS, name="loss_bf16_largest_train", N=16384, H=4096, V=100003, dtype="bfloat16"),
        # Perplexity of a document: every token's own loss, no gradient.
        dict(_LOSS, name="loss_bf16_score", N=2047, H=1024, V=50021, dtype="bfloat16", reduction="none", train=False),
        # Serving: the log probability of one sampled token, the head read once.
        dict(_LOSS, name="loss_one_token_score", N=1, H=4096, V=100003, dtype="bfloat16", reduction="none",
             train=False, ignored=0.0),
        # Decoding: the embeddings of eight requests' last tokens.
        dict(_EMBED, name="embed_decode", n=8, H=512, V=32000, scale=math.sqrt(512.0), train=False),
        # A float32 training batch of ordinary size.
        dict(_EMBED, name="embed_f32_train", n=16384, H=512, V=32000, scale=math.sqrt(512.0)),
        # The largest: a long batch with padded tails, a few tokens that are a tenth of the text each.
        dict(_EMBED, name="embed_bf16_train", n=131071, H=2048, V=100003, dtype="bfloat16", scale=math.sqrt(2048.0),
             pads=0.2),
        # The stack of a formal-language model between two healthy steps: the norm, and nothing to clip.
        dict(_CLIP, name="clip_small_in_place", blocks=4, H=32, V=8, clipped=False, in_place=True),
        # A float32 model of 0.29 billion parameters in 196 tensors, clipped.
        dict(_CLIP, name="clip_f32", blocks=24, H=1024, V=32000),
        # The largest: 3.2 billion parameters in bfloat16, clipped.
        dict(_CLIP, name="clip_bf16_largest", blocks=16, H=4096, V=100003, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    pick = rng.randrange(7)
    dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
    if pick <= 2:
        while True:
            N, H, V = _log(rng, 1, 16384), _log(rng, 32, 4096), _log(rng, 8, 100003)
            if rng.random() < 0.6:  # most models' widths are multiples of 64; the others stay as drawn
                H = max(64, H // 64 * 64)
            # a float32 multiply-add counts for eight of bfloat16's
            if N * H * V * (8 if dtype == "float32" else 1) <= LARGEST:
                break
        train = rng.random() < 0.7
        return dict(_LOSS, N=N, H=H, V=V, dtype=dtype, bias=rng.random() < 0.5,
                    reduction=rng.choice(["mean", "mean", "none"]), train=train,
                    ignored=0.0 if N < 4 else rng.choice([0.0, 0.1, 0.5]))
    if pick <= 4:
        while True:
            n, H, V = _log(rng, 1, 131071), _log(rng, 32, 4096), _log(rng, 8, 100003)
            if n * H <= LARGEST_ROWS and V * H <= LARGEST_TABLE:
                break
        return dict(_EMBED, n=n, H=H, V=V, dtype=dtype, scale=rng.choice([1.0, math.sqrt(H)]),
                    pads=rng.choice([0.0, 0.2, 0.5]), train=rng.random() < 0.7)
    while True:
        case = dict(_CLIP, blocks=_log(rng, 1, 48), H=_log(rng, 32, 4096), V=_log(rng, 8, 100003), dtype=dtype)
        if sum(math.prod(s) for s in _shapes(case)) <= LARGEST_GRADS // (2 if dtype == "float32" else 1):
            break
    in_place = rng.random() < 0.3
    return dict(case, in_place=in_place, clipped=not in_place and rng.random() < 0.8)


# ------------------------------------------------------------------------------------------------------ the inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _generator(case, seed):
    g = torch.Generator(device=_device())
    g.manual_seed(1000003 * int(seed) + 7919 * case["H"] + case["V"])
    return g


def _frequencies(V):
    """A text's token frequencies: the rank's reciprocal power."""
    p = 1.0 / (np.arange(V, dtype=np.float64) + 2.7)
    return p / p.sum()


def _tokens(n, V, g):
    cdf = torch.tensor(np.cumsum(_frequencies(V)), device=_device(), dtype=torch.float64)
    u = torch.rand(n, generator=g, device=_device(), dtype=torch.float64)
    ranks = torch.searchsorted(cdf, u).clamp_(max=V - 1)
    return torch.randperm(V, generator=g, device=_device())[ranks]  # frequent tokens anywhere in the vocabulary


def _shapes(case):
    """The shapes of a stack's gradients: embedding, per block two norms, the maps down, up and back, a gate; head."""
    H, V = case["H"], case["V"]
    out = [(V, H)]
    for _ in range(case["blocks"]):
        out += [(H,), (H,), (H, H), (H,), (4 * H, H), (4 * H,), (H, 4 * H), (H,)]
    return out + [(H,), (V, H), (V,)]


def prepare(case, seed):
    g = _generator(case, seed)
    dev = _device()
    state = dict(case)
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(0, PACKAGE)
        import ews_mi355x

        state["E"] = ews_mi355x
    if case["kind"] == "loss":
        state.update(_loss_inputs(case, g, dev))
    elif case["kind"] == "embed":
        state.update(_embed_inputs(case, g, dev))
    else:
        state.update(_clip_inputs(case, g, dev))
    return state


def _loss_inputs(case, g, dev):
    """Normalised hidden rows that lean towards their target's row of the head; logits of a few units."""
    N, H, V, dt = case["N"], case["H"], case["V"], DTYPES[case["dtype"]]
    weight = (torch.randn(V, H, generator=g, device=dev) * (1.5 / math.sqrt(H))).to(dt)
    targets = _tokens(N, V, g)
    lean = 4.0 * torch.rand(N, 1, generator=g, device=dev)
    hidden = (torch.randn(N, H, generator=g, device=dev) + lean * weight[targets].float()).to(dt)
    bias = (0.5 * torch.randn(V, generator=g, device=dev)).to(dt) if case["bias"] else None
    drop = torch.rand(N, generator=g, device=dev) < case["ignored"]
    targets = torch.where(drop, torch.full_like(targets, IGNORE), targets)
    upstream = torch.rand(N, generator=g, device=dev) + 0.5 if case["reduction"] == "none" else None
    if case["train"]:
        for t in (hidden, weight, bias):
            if t is not None:
                t.requires_grad_()
    return dict(hidden=hidden, weight=weight, bias=bias, targets=targets, upstream=upstream)


def _embed_inputs(case, g, dev):
    n, H, V, dt = case["n"], case["H"], case["V"], DTYPES[case["dtype"]]
    weight = (torch.randn(V, H, generator=g, device=dev) / math.sqrt(H)).to(dt)
    tokens = _tokens(n, V, g)
    pad = 0 if case["pads"] > 0 else None
    if pad is not None:
        tokens[n - int(case["pads"] * n):] = pad
    upstream = (torch.randn(n, H, generator=g, device=dev) * 1e-2).to(dt) if case["train"] else None
    if case["train"]:
        weight.requires_grad_()
    return dict(weight=weight, tokens=tokens, pad=pad, upstream=upstream)


def _in_one(shapes, dtype, dev):
    """Tensors of these shapes in one zeroed buffer, as a trainer that exchanges its gradients keeps them."""
    starts, end = [], 0
    for s in shapes:
        starts.append(end)
        end += -(-math.prod(s) // 64) * 64
    flat = torch.zeros(end, device=dev, dtype=dtype)
    return flat, [flat[a:a + math.prod(s)].view(s) for a, s in zip(starts, shapes)]


def _clip_inputs(case, g, dev):
    dt = DTYPES[case["dtype"]]
    shapes = _shapes(case)
    count = sum(math.prod(s) for s in shapes)
    flat, out = _in_one(shapes, dt, dev)
    grads = out if case["in_place"] else [torch.empty(s, device=dev, dtype=dt) for s in shapes]
    for i, t in enumerate(grads):
        t.normal_(generator=g).mul_(10.0 ** (-1 - i % 3) / math.sqrt(count))
    # the norm is a few hundredths: a bound of 0.001 clips, one of 1 does not
    state = dict(grads=grads, out=out, flat=flat, max_norm=0.001 if case["clipped"] else 1.0)
    if case["in_place"]:
        state["params"] = [torch.empty_like(t).requires_grad_() for t in grads]
        for p, t in zip(state["params"], grads):
            p.grad = t
    return state


# --------------------------------------------------------------------------------------------------------- one pass
def run(state):
    fn = {"loss": (_plain_loss, _own_loss), "embed": (_plain_embed, _own_embed), "clip": (_plain_clip, _own_clip)}
    return fn[state["kind"]][1 if own else 0](state)


def _own_loss(s):
    E = s["E"]
    if not s["train"]:
        with torch.no_grad():
            return E.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], bias=s["bias"],
                                          ignore_index=IGNORE, reduction=s["reduction"])
    loss = E.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], bias=s["bias"], ignore_index=IGNORE,
                                  reduction=s["reduction"])
    wrt = [t for t in (s["hidden"], s["weight"], s["bias"]) if t is not None]
    return (loss.detach(), *torch.autograd.grad(loss, wrt, s["upstream"]))


@torch.no_grad()
def _plain_loss(s):
    x, w = s["hidden"].float(), s["weight"].float()
    kept = s["targets"] != IGNORE
    t = torch.where(kept, s["targets"], torch.zeros_like(s["targets"]))
    z = x @ w.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    zt = z.gather(1, t[:, None])[:, 0]
    m = z.max(1, keepdim=True).values
    z -= m
    z.exp_()
    total = z.sum(1, keepdim=True)
    zero = torch.zeros_like(zt)
    rows = torch.where(kept, torch.log(total[:, 0]) + m[:, 0] - zt, zero)
    count = kept.sum().clamp(min=1).float()
    loss = rows if s["reduction"] == "none" else rows.sum() / count
    if not s["train"]:
        return loss
    up = s["upstream"] if s["reduction"] == "none" else torch.ones_like(zt) / count
    z /= total
    z.scatter_add_(1, t[:, None], torch.full_like(zt, -1.0)[:, None])
    z *= torch.where(kept, up, zero)[:, None]
    out = [loss, (z @ w).to(s["hidden"].dtype), (z.t() @ x).to(s["weight"].dtype)]
    if s["bias"] is not None:
        out.append(z.sum(0).to(s["bias"].dtype))
    return tuple(out)


def _own_embed(s):
    E = s["E"]
    if not s["train"]:
        with torch.no_grad():
            return E.embedding_lookup(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["pad"])
    out = E.embedding_lookup(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["pad"])
    return (out.detach(), *torch.autograd.grad(out, [s["weight"]], s["upstream"]))


@torch.no_grad()
def _plain_embed(s):
    w, t = s["weight"], s["tokens"]
    out = (w[t].float() * s["scale"]).to(w.dtype)
    if not s["train"]:
        return out
    g = s["upstream"].float() * s["scale"]
    if s["pad"] is not None:
        g = torch.where((t == s["pad"])[:, None], torch.zeros_like(g), g)
    grad = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
    grad.index_add_(0, t, g)
    return out, grad.to(w.dtype)


def _own_clip(s):
    if s["in_place"]:
        return s["E"].clip_grad_norm_(s["params"], s["max_norm"]), s["flat"]
    norm, _ = s["E"].clip_grads(s["grads"], s["max_norm"], out=s["out"])
    return norm, s["flat"]


@torch.no_grad()
def _plain_clip(s):
    total = None
    for t in s["grads"]:
        f = t.float()
        sq = (f * f).sum()
        total = sq if total is None else total + sq
    norm = torch.sqrt(total)
    coef = torch.clamp(s["max_norm"] / (norm + NORM_EPS), max=1.0)
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * coef)
    return norm, s["flat"]


# ------------------------------------------------------------------------------------------ the definition in 64 bits
@torch.no_grad()
def exact(case, seed):
    g = _generator(case, seed)
    dev = _device()
    if case["kind"] == "loss":
        return _exact_loss(case, _loss_inputs(case, g, dev))
    if case["kind"] == "embed":
        return _exact_embed(case, _embed_inputs(case, g, dev))
    s = _clip_inputs(case, g, dev)
    squares = [torch.linalg.vector_norm(t.detach(), dtype=torch.float64) ** 2 for t in s["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    factor = min(1.0, s["max_norm"] / (float(norm) + NORM_EPS))
    flat, out = _in_one([t.shape for t in s["grads"]], torch.float64, dev)
    for t, o in zip(s["grads"], out):
        o.copy_(t.double() * factor)
    return norm, flat


def _exact_loss(case, s):
    N, V = case["N"], case["V"]
    x, w = s["hidden"].detach().double(), s["weight"].detach().double()
    b = None if s["bias"] is None else s["bias"].detach().double()
    t = s["targets"]
    valid = int((t != IGNORE).sum())
    loss = torch.zeros(N, device=x.device, dtype=torch.float64)
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    gb = None if b is None else torch.zeros_like(b)
    step = max(1, min(N, (1 << 28) // V))
    for lo in range(0, N, step):
        rows = torch.nonzero(t[lo:lo + step] != IGNORE)[:, 0] + lo
        if rows.numel() == 0:
            continue
        xr = x[rows]
        z = torch.matmul(xr, w.t()) if b is None else torch.addmm(b, xr, w.t())
        logp = torch.log_softmax(z, 1)
        del z
        loss[rows] = -logp[torch.arange(rows.numel(), device=x.device), t[rows]]
        if not case["train"]:
            continue
        d = logp.exp_()
        d[torch.arange(rows.numel(), device=x.device), t[rows]] -= 1.0
        d *= s["upstream"].double()[rows][:, None] if case["reduction"] == "none" else 1.0 / valid
        gx[rows] = torch.matmul(d, w)
        gw += torch.matmul(d.t(), xr)
        if gb is not None:
            gb += d.sum(0)
    value = loss if case["reduction"] == "none" else loss.sum() / max(1, valid)
    if not case["train"]:
        return value
    return (value, gx, gw) if gb is None else (value, gx, gw, gb)


def _exact_embed(case, s):
    w, t = s["weight"].detach().double(), s["tokens"]
    out = w.index_select(0, t) * case["scale"]
    if not case["train"]:
        return out
    keep = torch.ones_like(t, dtype=torch.bool) if s["pad"] is None else t != s["pad"]
    grad = torch.zeros_like(w).index_add_(0, t[keep], s["upstream"].double()[keep])
    return out, grad * case["scale"]


# ------------------------------------------------------------------------------------------------------------ the work
def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "loss":
        N, H, V = case["N"], case["H"], case["V"]
        b = V * e if case["bias"] else 0
        rows = N if case["reduction"] == "none" else 0
        read = (N * H + V * H) * e + b + 8 * N
        if not case["train"]:
            return {"bytes": read + 4 * max(1, rows), "flops": 2 * N * V * H}
        return {"bytes": read + 4 * rows + 4 * max(1, rows) + (N * H + V * H) * e + b, "flops": 6 * N * V * H}
    if case["kind"] == "embed":
        n, H, V = case["n"], case["H"], case["V"]
        live = n - int(case["pads"] * n)
        distinct = float((1.0 - (1.0 - _frequencies(V)) ** live).sum())
        moved = 8 * n + (n + distinct) * H * e
        if case["train"]:
            moved += (live + V) * H * e
        return {"bytes": int(moved), "flops": n * H + (live * H if case["train"] else 0)}
    count = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": count * e * (1 if case["in_place"] else 2), "flops": 2 * count + (count if case["clipped"] else 0)}
