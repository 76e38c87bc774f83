"""Trains a small token model to predict the next token of a synthetic language: after token t comes t + 1 nine times in
ten (modulo the vocabulary), else any.

One step is the whole of a language model's: embedding lookup, EWS blocks, the head's cross entropy without the logits
in memory (``StackedEWS.loss``), backward, clipping by the gradients' global norm (``clip_grad_norm_``), AdamW.

    python examples/train_tokens.py [--steps 200] [--batch 64] [--length 64] [--base 16]
"""

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "exponentially-weighted-signature_amd")
if PACKAGE not in sys.path:
    sys.path.insert(0, PACKAGE)

import ews_mi355x as E  # noqa: E402


def batch(n, length, base, g):
    """Tokens 1..base (0 pads ragged ends), the next ones as classes 0..base-1, and the mask of real positions."""
    rest = torch.rand(n, length + 1, generator=g) < 0.1
    anyone = torch.randint(0, base, (n, length + 1), generator=g)
    text = torch.empty(n, length + 1, dtype=torch.int64)
    text[:, 0] = anyone[:, 0]
    for k in range(1, length + 1):
        text[:, k] = torch.where(rest[:, k], anyone[:, k], (text[:, k - 1] + 1) % base)
    ends = torch.randint(length // 2, length + 1, (n,), generator=g)
    mask = torch.arange(length)[None] < ends[:, None]
    return (text[:, :-1] + 1).masked_fill(~mask, 0).cuda(), text[:, 1:].cuda(), mask.cuda()


def make_model(base, hidden=32, blocks=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    rates = [dict(a_param=E.AParamDampedRotation(torch.randn(hidden // 2, generator=g) - 4.0,
                                                 torch.randn(hidden // 2, generator=g), hidden))
             for _ in range(blocks)]
    kwargs = dict(m=hidden, n=1, leaf="plane_closed", combine="block_kernel", basepoint=True, channel_stage="glu",
                  path_mode="increment", dropout_rate=0.0)
    return E.StackedEWS(blocks, base + 1, hidden, base, tokens=True, block_kwargs=kwargs, per_block_kwargs=rates,
                        key=seed).cuda()


def train(steps=200, n=64, length=64, base=16, max_norm=1.0, lr=3e-3, seed=0, report=None):
    """The losses of every step; report(step, loss, norm) is called with device numbers."""
    g = torch.Generator().manual_seed(seed)
    model = make_model(base, seed=seed)
    opt = torch.optim.AdamW(model.parameters(), lr=lr, weight_decay=0.0)
    losses = []
    for step in range(steps):
        tokens, targets, mask = batch(n, length, base, g)
        loss = model.loss(tokens, targets, mask=mask)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        norm = E.clip_grad_norm_(model.parameters(), max_norm)
        opt.step()
        losses.append(loss.detach())
        if report is not None:
            report(step, losses[-1], norm)
    return torch.stack(losses)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--length", type=int, default=64)
    ap.add_argument("--base", type=int, default=16)
    args = ap.parse_args()

    def report(step, loss, norm):
        if step % 20 == 0 or step + 1 == args.steps:
            print(f"step {step:4d}  loss {float(loss):.4f}  gradient norm {float(norm):.3f}", flush=True)

    train(args.steps, args.batch, args.length, args.base, report=report)


if __name__ == "__main__":
    main()
