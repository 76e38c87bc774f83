"""What is timed of the operators inside a token model's blocks and of its training from a teacher: the gated linear
map of a channel stage, the gated linear recurrence over a sequence, and the distillation loss from a teacher's top
logits.

Every case runs one whole call on inputs made from the seed. Where ``own`` is false ``run`` computes the operator in
its plain form with elementary torch operations in float32, rounded once at the end; where it is true ``run`` calls
the package. ``exact`` restates the definition in float64.

Kinds of case:

    gated    ``gated_linear`` of N rows of width H to F gated results
    scan     ``gated_scan`` of B sequences of L steps and D channels
    distill  ``linear_distillation`` of N rows of width H, a vocabulary of V and K teacher's entries a row
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "exponentially-weighted-signature_amd")

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}

_GATED = dict(kind="gated", N=1, H=1, F=1, dtype="float32", activation="sigmoid", joint=True, bias=True, train=True)
_SCAN = dict(kind="scan", B=1, L=1, D=1, dtype="float32", form="convex", ragged=False, state=True, train=True)
_DISTILL = dict(kind="distill", N=1, H=1, V=1, K=1, dtype="float32", bias=False, temperature=1.0, reduction="mean",
                padded=0.1, train=True)

LARGEST_GATED = 16384 * 4096 * 11000  # N H F
LARGEST_SCAN = 131071 * 1024  # B L D
LARGEST_DISTILL = 2 * LARGEST_GATED  # N H V: half the products of a gated row


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # Decoding: one token through a wide channel stage, the weights read once.
        dict(_GATED, name="gated_decode", N=1, H=4096, F=11000, dtype="bfloat16", activation="silu", joint=False,
             bias=False, train=False),
        # The channel stage of a formal-language stack: 256 sequences of 512 tokens, width 32.
        dict(_GATED, name="gated_narrow_f32_train", N=131072, H=32, F=32),
        # A float32 model of the package's default type, odd row count.
        dict(_GATED, name="gated_f32_train", N=4095, H=512, F=1365, activation="gelu"),
        # A bfloat16 training step of ordinary size.
        dict(_GATED, name="gated_bf16_train", N=8192, H=2048, F=5504, dtype="bfloat16", activation="silu", joint=False,
             bias=False),
        # The largest: a wide model on a long batch, a width that no tile divides.
        dict(_GATED, name="gated_bf16_largest_train", N=16384, H=4096, F=11000, dtype="bfloat16", activation="silu",
             bias=False),
        # Decoding: one step of eight requests.
        dict(_SCAN, name="scan_decode", B=8, L=1, D=2048, dtype="bfloat16", train=False),
        # A regression model on very long series, width 24.
        dict(_SCAN, name="scan_narrow_f32_train", B=8, L=49920, D=24, form="linear", state=False),
        # A bfloat16 training batch of padded texts.
        dict(_SCAN, name="scan_bf16_train", B=8, L=4095, D=2048, dtype="bfloat16", ragged=True, state=False),
        # The largest: one long document with a state carried over from the part before.
        dict(_SCAN, name="scan_long_bf16_train", B=1, L=131071, D=1024, dtype="bfloat16"),
        # A small student on a short batch: launches and their latency are most of it.
        dict(_DISTILL, name="distill_small_f32_train", N=256, H=64, V=1000, K=8, bias=True, temperature=2.0),
        # A bfloat16 training step of ordinary size.
        dict(_DISTILL, name="distill_bf16_train", N=8192, H=2048, V=32000, K=32, dtype="bfloat16", temperature=2.0),
        # How far a student is from its teacher on a document: every token's own loss, no gradient.
        dict(_DISTILL, name="distill_bf16_score", N=2047, H=1024, V=50021, K=100, dtype="bfloat16", reduction="none",
             train=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    pick = rng.randrange(3)
    dtype = rng.choice(["float32", "bfloat16", "bfloat16"])
    slow = 8 if dtype == "float32" else 1  # a float32 multiply-add counts for eight of bfloat16's
    train = rng.random() < 0.7
    if pick == 0:
        while True:
            N, H, F = _log(rng, 1, 131072), _log(rng, 32, 4096), _log(rng, 32, 16384)
            if rng.random() < 0.6:  # most models' widths are multiples of 64; the others stay as drawn
                H, F = max(64, H // 64 * 64), max(64, F // 64 * 64)
            if N * H * F * slow <= LARGEST_GATED and N * max(H, F) <= 1 << 28:
                break
        return dict(_GATED, N=N, H=H, F=F, dtype=dtype, activation=rng.choice(["sigmoid", "silu", "gelu", "relu"]),
                    joint=rng.random() < 0.5, bias=rng.random() < 0.5, train=train)
    if pick == 1:
        while True:
            B, L, D = _log(rng, 1, 256), _log(rng, 1, 131071), _log(rng, 8, 4096)
            if rng.random() < 0.6:
                D = max(16, D // 16 * 16)
            if B * L * D <= LARGEST_SCAN:
                break
        return dict(_SCAN, B=B, L=L, D=D, dtype=dtype, form=rng.choice(["convex", "convex", "linear"]),
                    ragged=rng.random() < 0.4, state=rng.random() < 0.5, train=train)
    while True:
        N, H, V = _log(rng, 1, 16384), _log(rng, 32, 4096), _log(rng, 8, 100003)
        if rng.random() < 0.6:
            H = max(64, H // 64 * 64)
        if N * H * V * slow <= LARGEST_DISTILL:
            break
    return dict(_DISTILL, N=N, H=H, V=V, K=_log(rng, 1, min(V, 256)), dtype=dtype, bias=rng.random() < 0.5,
                temperature=rng.choice([1.0, 1.0, 2.0, 4.0]), reduction=rng.choice(["mean", "mean", "none"]),
                padded=0.0 if N < 4 else rng.choice([0.0, 0.1, 0.5]), train=train)


# ------------------------------------------------------------------------------------------------------ the inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _generator(case, seed):
    g = torch.Generator(device=_device())
    sizes = [v for v in case.values() if isinstance(v, int)]
    g.manual_seed(1000003 * int(seed) + 7919 * max(sizes) + sum(sizes))
    return g


def prepare(case, seed):
    state = dict(case)
    if own:
        if PACKAGE not in sys.path:
            sys.path.insert(0, PACKAGE)
        import ews_mi355x

        state["E"] = ews_mi355x
    state.update(_inputs(case, seed))
    return state


def _inputs(case, seed):
    make = {"gated": _gated_inputs, "scan": _scan_inputs, "distill": _distill_inputs}[case["kind"]]
    return make(case, _generator(case, seed), _device())


def _wants(case, tensors):
    if case["train"]:
        for t in tensors:
            if t is not None:
                t.requires_grad_()


def _gated_inputs(case, g, dev):
    """Normalised rows, maps of the usual initial size, biases of the same order, an upstream of a loss's mean."""
    N, H, F, dt = case["N"], case["H"], case["F"], DTYPES[case["dtype"]]

    def weight(rows):
        return (torch.randn(rows, H, generator=g, device=dev) / math.sqrt(H)).to(dt)

    def bias(rows):
        return (0.3 * torch.randn(rows, generator=g, device=dev)).to(dt) if case["bias"] else None

    x = torch.randn(N, H, generator=g, device=dev).to(dt)
    if case["joint"]:
        w, b, gw, gb = weight(2 * F), bias(2 * F), None, None
    else:
        w, b, gw, gb = weight(F), bias(F), weight(F), bias(F)
    upstream = (0.02 * torch.randn(N, F, generator=g, device=dev)).to(dt) if case["train"] else None
    _wants(case, (x, w, b, gw, gb))
    return dict(x=x, weight=w, bias_=b, gate_weight=gw, gate_bias=gb, upstream=upstream)


def _scan_inputs(case, g, dev):
    """Gates that remember a few tokens to some hundreds; ragged texts padded at their end."""
    B, L, D, dt = case["B"], case["L"], case["D"], DTYPES[case["dtype"]]
    x = torch.randn(B, L, D, generator=g, device=dev).to(dt)
    gate = torch.randn(B, L, D, generator=g, device=dev) + 4.0 * torch.rand(D, generator=g, device=dev)
    gate = gate.to(dt) if case["form"] == "convex" else torch.sigmoid(gate).to(dt)
    mask = None
    if case["ragged"]:
        lengths = torch.randint(L // 2, L + 1, (B, 1), generator=g, device=dev)
        mask = torch.arange(L, device=dev)[None] < lengths
    state = torch.randn(B, D, generator=g, device=dev) if case["state"] else None
    out = dict(x=x, gate=gate, mask=mask, state0=state)
    if case["train"]:
        out["upstream"] = (0.02 * torch.randn(B, L, D, generator=g, device=dev)).to(dt)
        out["upstream_last"] = 0.02 * torch.randn(B, D, generator=g, device=dev)
    else:
        out["last"] = torch.empty(B, D, device=dev)
    _wants(case, (x, gate, state))
    return out


def _distill_inputs(case, g, dev):
    """A teacher that agrees with the student's lean on some tokens: its K largest logits, in falling order, at tokens
    that differ; some rows (padding) have none, others fewer than K."""
    N, H, V, K, dt = case["N"], case["H"], case["V"], case["K"], DTYPES[case["dtype"]]
    weight = (torch.randn(V, H, generator=g, device=dev) * (1.5 / math.sqrt(H))).to(dt)
    # K different tokens: a stretch of a random order from a random place on, frequent ones anywhere
    order = torch.randperm(V, generator=g, device=dev)
    start = torch.randint(0, V, (N, 1), generator=g, device=dev)
    indices = order[(start + torch.arange(K, device=dev)) % V]
    lean = 4.0 * torch.rand(N, 1, generator=g, device=dev)
    hidden = (torch.randn(N, H, generator=g, device=dev) + lean * weight[indices[:, 0]].float()).to(dt)
    logits = torch.sort(3.0 * torch.randn(N, K, generator=g, device=dev), dim=1, descending=True).values
    used = torch.randint(1, K + 1, (N, 1), generator=g, device=dev)
    used = torch.where(torch.rand(N, 1, generator=g, device=dev) < 0.2, used, torch.full_like(used, K))
    used = torch.where(torch.rand(N, 1, generator=g, device=dev) < case["padded"], torch.zeros_like(used), used)
    indices = torch.where(torch.arange(K, device=dev) < used, indices, torch.full_like(indices, -1))
    bias = (0.5 * torch.randn(V, generator=g, device=dev)).to(dt) if case["bias"] else None
    upstream = torch.rand(N, generator=g, device=dev) + 0.5 if case["reduction"] == "none" else None
    _wants(case, (hidden, weight, bias))
    return dict(hidden=hidden, weight=weight, bias_=bias, indices=indices, logits=logits, upstream=upstream)


# --------------------------------------------------------------------------------------------------------- one pass
def run(state):
    fn = {"gated": (_plain_gated, _own_gated), "scan": (_plain_scan, _own_scan),
          "distill": (_plain_distill, _own_distill)}
    return fn[state["kind"]][1 if own else 0](state)


def _given(*tensors):
    return [t for t in tensors if t is not None]


def _own_gated(s):
    E = s["E"]
    args = dict(bias=s["bias_"], gate_weight=s["gate_weight"], gate_bias=s["gate_bias"], activation=s["activation"])
    if not s["train"]:
        with torch.no_grad():
            return E.gated_linear(s["x"], s["weight"], **args)
    y = E.gated_linear(s["x"], s["weight"], **args)
    wrt = _given(s["x"], s["weight"], s["bias_"], s["gate_weight"], s["gate_bias"])
    return (y.detach(), *torch.autograd.grad(y, wrt, s["upstream"]))


def _own_scan(s):
    E = s["E"]
    if not s["train"]:
        with torch.no_grad():
            return E.gated_scan(s["x"], s["gate"], state=s["state0"], mask=s["mask"], form=s["form"], last=s["last"])
    h, last = E.gated_scan(s["x"], s["gate"], state=s["state0"], mask=s["mask"], form=s["form"])
    wrt = _given(s["x"], s["gate"], s["state0"])
    return (h.detach(), last.detach(), *torch.autograd.grad((h, last), wrt, (s["upstream"], s["upstream_last"])))


def _own_distill(s):
    E = s["E"]
    args = dict(bias=s["bias_"], temperature=s["temperature"], reduction=s["reduction"])
    if not s["train"]:
        with torch.no_grad():
            return E.linear_distillation(s["hidden"], s["weight"], s["indices"], s["logits"], **args)
    loss = E.linear_distillation(s["hidden"], s["weight"], s["indices"], s["logits"], **args)
    wrt = _given(s["hidden"], s["weight"], s["bias_"])
    return (loss.detach(), *torch.autograd.grad(loss, wrt, s["upstream"]))


# --------------------------------------------------------------------------------------------------- the plain forms
_GELU_A, _GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def _activate(g, name):
    """act(g) and its derivative."""
    if name == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if name == "gelu":
        t = torch.tanh(_GELU_A * (g + _GELU_B * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * _GELU_A * (1 + 3 * _GELU_B * g * g)
    p = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return p, p * (1 - p)
    return g * p, p * (1 + g * (1 - p))


@torch.no_grad()
def _plain_gated(s):
    dt, F, joint = s["x"].dtype, s["F"], s["gate_weight"] is None
    x, w = s["x"].float(), s["weight"].float()
    wv, wg = (w[:F], w[F:]) if joint else (w, s["gate_weight"].float())
    v, g = x @ wv.t(), x @ wg.t()
    if s["bias_"] is not None:
        b = s["bias_"].float()
        v += b[:F]
        g += b[F:] if joint else s["gate_bias"].float()
    act, slope = _activate(g, s["activation"])
    y = (v * act).to(dt)
    if not s["train"]:
        return y
    up = s["upstream"].float()
    dv, dg = up * act, up * v * slope
    del v, g, act, slope
    dx = (dv @ wv + dg @ wg).to(dt)
    dw = [dv.t() @ x, dg.t() @ x]
    db = [dv.sum(0), dg.sum(0)] if s["bias_"] is not None else None
    if joint:
        out = [y, dx, torch.cat(dw).to(dt)]
        return tuple(out if db is None else out + [torch.cat(db).to(dt)])
    if db is None:
        return y, dx, dw[0].to(dt), dw[1].to(dt)
    return y, dx, dw[0].to(dt), db[0].to(dt), dw[1].to(dt), db[1].to(dt)


def _doubling(a, b):
    """Every h_t = a_t h_{t-1} + b_t (dim 1) from h = 0, and the products of the a up to each t, by doubling."""
    a, b = a.clone(), b.clone()
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return a, b


@torch.no_grad()
def _plain_scan(s):
    dt, convex = s["x"].dtype, s["form"] == "convex"
    x, g = s["x"].float(), s["gate"].float()
    a = 1.0 / (1.0 + torch.exp(-g)) if convex else g
    take = 1.0 / (1.0 + torch.exp(g)) if convex else torch.ones_like(a)  # 1 - a without its rounding
    b = take * x
    if s["mask"] is not None:
        off = ~s["mask"][..., None]
        a, b, take = a.masked_fill(off, 1.0), b.masked_fill(off, 0.0), take.masked_fill(off, 0.0)
    total, h = _doubling(a, b)
    h0 = s["state0"]
    h0 = torch.zeros_like(h[:, 0]) if h0 is None else h0
    h = h + total * h0[:, None]
    del total, b
    if not s["train"]:
        return h.to(dt), h[:, -1].clone()
    up = s["upstream"].float().clone()  # float32 too: the state keeps its own
    up[:, -1] += s["upstream_last"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    _, lam = _doubling(after.flip(1), up.flip(1))
    lam = lam.flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    slope = (before - x) * a * take if convex else before
    if s["mask"] is not None:
        slope = slope.masked_fill(off, 0.0)
    out = [h.to(dt), h[:, -1].clone(), (lam * take).to(dt), (lam * slope).to(dt)]
    if s["state0"] is not None:
        out.append(lam[:, 0] * a[:, 0])
    return tuple(out)


@torch.no_grad()
def _plain_distill(s):
    x, w, T = s["hidden"].float(), s["weight"].float(), s["temperature"]
    has = s["indices"] >= 0
    at = torch.where(has, s["indices"], torch.zeros_like(s["indices"]))
    kept = has.any(1)
    u = torch.where(has, s["logits"].float() / T, torch.full_like(s["logits"], -math.inf))
    top = torch.where(kept[:, None], u.max(1, keepdim=True).values, torch.zeros_like(u[:, :1]))
    e = torch.where(has, torch.exp(u - top), torch.zeros_like(u))
    total = e.sum(1, keepdim=True).clamp(min=1e-30)
    p = e / total
    logp = torch.where(has, u - top - torch.log(total), torch.zeros_like(u))
    z = x @ w.t()
    if s["bias_"] is not None:
        z += s["bias_"].float()
    z /= T
    m = z.max(1, keepdim=True).values
    zk = z.gather(1, at) - m
    z -= m
    z.exp_()
    total = z.sum(1, keepdim=True)
    rows = T * T * (p * (logp - zk + torch.log(total))).sum(1)
    rows = torch.where(kept, rows, torch.zeros_like(rows))
    count = kept.sum().clamp(min=1).float()
    loss = rows if s["reduction"] == "none" else rows.sum() / count
    if not s["train"]:
        return loss
    up = s["upstream"] if s["reduction"] == "none" else torch.ones_like(rows) / count
    z /= total
    z.scatter_add_(1, at, -p)
    z *= torch.where(kept, T * up, torch.zeros_like(up))[:, None]
    out = [loss, (z @ w).to(s["hidden"].dtype), (z.t() @ x).to(s["weight"].dtype)]
    if s["bias_"] is not None:
        out.append(z.sum(0).to(s["bias_"].dtype))
    return tuple(out)


# ------------------------------------------------------------------------------------------ the definition in 64 bits
@torch.no_grad()
def exact(case, seed):
    s = _inputs(case, seed)
    return {"gated": _exact_gated, "scan": _exact_scan, "distill": _exact_distill}[case["kind"]](case, s)


def _double(t):
    return None if t is None else t.detach().double()


def _exact_activation(g, name):
    if name == "relu":
        return torch.where(g > 0, g, 0.0), torch.where(g > 0, 1.0, 0.0).to(g.dtype)
    if name == "gelu":  # g sigmoid(2 u), u = sqrt(2 / pi) (g + 0.044715 g^3): the same function as with tanh
        inner = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)
        p = torch.sigmoid(inner)
        return g * p, p + g * p * torch.sigmoid(-inner) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * g**2)
    p, q = torch.sigmoid(g), torch.sigmoid(-g)
    return (p, p * q) if name == "sigmoid" else (g * p, p + g * p * q)


def _exact_gated(case, s):
    F, train = case["F"], case["train"]
    x, w, b, gw, gb = (_double(s[k]) for k in ("x", "weight", "bias_", "gate_weight", "gate_bias"))
    joint = gw is None
    w = w if joint else torch.cat([w, gw])
    b = b if joint or b is None else torch.cat([b, gb])
    y = torch.empty(case["N"], F, device=x.device, dtype=torch.float64)
    dx, dw = (torch.zeros_like(x), torch.zeros_like(w)) if train else (None, None)
    db = torch.zeros(2 * F, device=x.device, dtype=torch.float64)
    step = max(1, (1 << 27) // F)
    for lo in range(0, case["N"], step):
        xs = x[lo:lo + step]
        z = torch.nn.functional.linear(xs, w, b)
        act, slope = _exact_activation(z[:, F:], case["activation"])
        y[lo:lo + step] = z[:, :F] * act
        if not train:
            continue
        u = _double(s["upstream"][lo:lo + step])
        dz = torch.cat([u * act, u * z[:, :F] * slope], 1)
        dx[lo:lo + step] = torch.matmul(dz, w)
        dw += torch.matmul(dz.t(), xs)
        db += dz.sum(0)
    if not train:
        return y
    if joint:
        return (y, dx, dw) if b is None else (y, dx, dw, db)
    if b is None:
        return y, dx, dw[:F], dw[F:]
    return y, dx, dw[:F], db[:F], dw[F:], db[F:]


def _steps(a, b, h):
    """Every h_t = a_t h_{t-1} + b_t (dim 1): chunks side by side step by step, then their ends one after another."""
    B, L, D = b.shape
    T = max(1, math.isqrt(L))
    C = -(-L // T)
    pad = C * T - L
    a = torch.nn.functional.pad(a, (0, 0, 0, pad), value=1.0).view(B, C, T, D)
    out = torch.nn.functional.pad(b, (0, 0, 0, pad)).view(B, C, T, D).clone()
    reach = a.clone()
    for t in range(1, T):
        out[:, :, t] += a[:, :, t] * out[:, :, t - 1]
        reach[:, :, t] *= reach[:, :, t - 1]
    for c in range(C):
        out[:, c] += reach[:, c] * h[:, None]
        h = out[:, c, -1].clone()
    return out.view(B, C * T, D)[:, :L]


def _exact_scan(case, s):
    x, g, h0 = _double(s["x"]), _double(s["gate"]), _double(s["state0"])
    convex = case["form"] == "convex"
    a, take = (torch.sigmoid(g), torch.sigmoid(-g)) if convex else (g.clone(), torch.ones_like(g))
    if s["mask"] is not None:
        off = ~s["mask"]
        a[off], take[off] = 1.0, 0.0
    start = torch.zeros_like(x[:, 0]) if h0 is None else h0
    h = _steps(a, take * x, start)
    if not case["train"]:
        return h, h[:, -1]
    up = _double(s["upstream"])
    up[:, -1] += _double(s["upstream_last"])
    lam = _steps(torch.cat([a[:, 1:], a[:, :1]], 1).flip(1), up.flip(1), torch.zeros_like(start)).flip(1)
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    dg = lam * before if not convex else lam * (before - x) * a * take
    if s["mask"] is not None:
        dg[off] = 0.0
    out = (h, h[:, -1], lam * take, dg)
    return out if h0 is None else (*out, lam[:, 0] * a[:, 0])


def _exact_distill(case, s):
    N, V, T = case["N"], case["V"], case["temperature"]
    x, w, b = _double(s["hidden"]), _double(s["weight"]), _double(s["bias_"])
    kept = (s["indices"] >= 0).any(1)
    count = max(1, int(kept.sum()))
    loss = torch.zeros(N, device=x.device, dtype=torch.float64)
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    gb = None if b is None else torch.zeros_like(b)
    step = max(1, min(N, (1 << 28) // V))
    for lo in range(0, N, step):
        rows = torch.nonzero(kept[lo:lo + step])[:, 0] + lo
        if rows.numel() == 0:
            continue
        index = s["indices"][rows]
        teacher = _double(s["logits"])[rows].masked_fill(index < 0, -math.inf)
        logp = torch.log_softmax(teacher / T, 1)
        p = logp.exp()
        xr = x[rows]
        logq = torch.nn.functional.linear(xr, w, b).div_(T)
        logq = torch.log_softmax(logq, 1)
        index = index.clamp(min=0)
        each = p * (logp - logq.gather(1, index))
        loss[rows] = T * T * torch.where(p > 0, each, 0.0).sum(1)
        if not case["train"]:
            continue
        d = logq.exp_()
        d.scatter_add_(1, index, -p)
        d *= T * s["upstream"].double()[rows][:, None] if case["reduction"] == "none" else T / count
        gx[rows] = torch.matmul(d, w)
        gw += torch.matmul(d.t(), xr)
        if gb is not None:
            gb += d.sum(0)
    value = loss if case["reduction"] == "none" else loss.sum() / count
    if not case["train"]:
        return value
    return (value, gx, gw) if gb is None else (value, gx, gw, gb)


# ------------------------------------------------------------------------------------------------------------ the work
def work(case):
    e, train = BYTES[case["dtype"]], case["train"]
    if case["kind"] == "gated":
        N, H, F = case["N"], case["H"], case["F"]
        params = 2 * F * H + (2 * F if case["bias"] else 0)
        moved = (N * H + params + N * F) * e
        if train:
            moved += (N * F + N * H + params) * e
        return {"bytes": moved, "flops": 4 * N * H * F * (3 if train else 1)}
    if case["kind"] == "scan":
        B, L, D = case["B"], case["L"], case["D"]
        n, ends = B * L * D, B * D * 4 * (2 if case["state"] else 1)
        moved = 3 * n * e + ends + (B * L if case["ragged"] else 0)
        if train:
            moved += 3 * n * e + ends
        return {"bytes": moved, "flops": n * (4 + (8 if train else 0))}
    N, H, V, K = case["N"], case["H"], case["V"], case["K"]
    b = V * e if case["bias"] else 0
    rows = N if case["reduction"] == "none" else 0
    moved = (N * H + V * H) * e + b + 12 * N * K + 4 * max(1, rows)
    if train:
        moved += 4 * rows + (N * H + V * H) * e + b
    return {"bytes": moved, "flops": 2 * N * V * H * (3 if train else 1)}
