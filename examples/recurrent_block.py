#!/usr/bin/env python
"""A stack of gated recurrent blocks, trained from activations kept in 8 bits, and served.

    python examples/recurrent_block.py [--width 256] [--blocks 2] [--tokens 1024] [--steps 20]

One block: the norm of the residual stream, a projection to values, gates of the
recurrence and an output gate, the recurrence of every channel (GatedRecurrence),
and what joins its output to the stream and makes the next block's input
(BlockNorm): norm, gate, scaled sum, norm.

* Training: packed sequences of different lengths.  The forward pass keeps what
  the backward passes need in 8 bits (Rows8) while it holds it; plain gradient
  descent on the distance to a teacher's outputs.
* Serving: packed prompts leave their states in slots; then single tokens of all
  requests at once.  Checked against the whole sequences run as one prompt.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from tensoroperations_b200 import sequence  # noqa: E402


class Stack:
    def __init__(self, width: int, blocks: int, dtype=torch.bfloat16, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.width, self.blocks, self.dtype = width, blocks, dtype
        normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.first = torch.ones(width, device="cuda")  # weight of the first norm
        self.w_in = [normal(width, 3 * width) / width ** 0.5 for _ in range(blocks)]
        self.bias = [1 + 4 * torch.rand(width, generator=gen, device="cuda") for _ in range(blocks)]
        self.w_post = [torch.ones(width, device="cuda") for _ in range(blocks)]
        self.w_pre = [torch.ones(width, device="cuda") for _ in range(blocks)]
        self.recurrence = sequence.GatedRecurrence(dtype, width)
        self.norm = sequence.BlockNorm(dtype, width, residual="f32", gate="silu", scale=0.5)

    def parameters(self):
        return [self.first, *self.w_in, *self.bias, *self.w_post, *self.w_pre]

    def _rows(self, n, w):
        rows = n @ w.to(self.dtype)
        return rows, rows[:, :self.width], rows[:, self.width:2 * self.width], rows[:, 2 * self.width:]

    def _new(self, t, kind=None):
        return torch.empty(t, self.width, dtype=kind or self.dtype, device="cuda")

    def forward(self, x, cu_seqlens, states=None, slots=None, kept=None):
        """The last norm's outputs; `kept` (a list) takes what the backward pass needs."""
        t, n = x.shape[0], cu_seqlens.numel() - 1
        ws = torch.empty(self.recurrence.workspace_bytes(t, n), dtype=torch.uint8, device="cuda")
        r, y = x.float(), self._new(t)
        keep = lambda: sequence.Rows8.empty(t, self.width) if kept is not None else None  # noqa: E731
        of = dict(r=keep())
        self.norm.forward(r, None, None, None, self.first, None, y, keep_r=of["r"])
        if kept is not None:
            kept.append(of)
        for b in range(self.blocks):
            of = dict(n=y, x=keep(), f=keep(), r=keep(), y=keep(), g=keep(), saved=None)
            _, v, f, g = self._rows(y, self.w_in[b])
            if kept is not None:
                of["saved"] = torch.empty(self.recurrence.saved_rows(t, n), self.width, device="cuda")
                kept.append(of)
            h, y, ro = self._new(t), self._new(t), self._new(t, torch.float32)
            state = None if states is None else states[b]
            self.recurrence.forward(v, f, self.bias[b], cu_seqlens, h, state_in=state, state_out=state, slots=slots,
                                    saved=of["saved"], keep_x=of["x"], keep_f=of["f"], workspace=ws)
            self.norm.forward(r, h, g, self.w_post[b], self.w_pre[b], ro, y, keep_r=of["r"], keep_y=of["y"], keep_g=of["g"])
            r = ro
        return y

    def token(self, x, states, slots=None):
        """One token of each request."""
        t = x.shape[0]
        r, y = x.float(), self._new(t)
        self.norm.forward(r, None, None, None, self.first, None, y)
        for b in range(self.blocks):
            _, v, f, g = self._rows(y, self.w_in[b])
            h, y = self._new(t), self._new(t)
            self.recurrence.step(v, f, self.bias[b], states[b], h, slots=slots)
            self.norm.forward(r, h, g, self.w_post[b], self.w_pre[b], r, y)
        return y

    def backward(self, dy, cu_seqlens, kept):
        """Gradients of the parameters, in their order, from that of the outputs."""
        t, n, w = dy.shape[0], cu_seqlens.numel() - 1, self.width
        ws = torch.empty(max(self.recurrence.backward_workspace_bytes(t, n), self.norm.workspace_bytes(t)),
                         dtype=torch.uint8, device="cuda")
        grads = {k: [None] * self.blocks for k in ("w_in", "bias", "w_post", "w_pre")}
        dr, dn = None, dy
        for b in reversed(range(self.blocks)):
            of = kept[b + 1]
            new, dh = self._new(t, torch.float32), self._new(t)
            rows = torch.empty(t, 3 * w, dtype=self.dtype, device="cuda")  # gradients of the projection's rows
            dw_post, dw_pre, dbias = (torch.empty(w, device="cuda") for _ in range(3))
            self.norm.backward(of["r"], of["y"], of["g"], self.w_post[b], self.w_pre[b], dr, dn, new, dh, rows[:, 2 * w:],
                               dw_post, dw_pre, ws)
            self.recurrence.backward(of["x"], of["f"], self.bias[b], cu_seqlens, of["saved"], dh, rows[:, :w], rows[:, w:2 * w],
                                     dbias, workspace=ws)
            grads["w_in"][b], grads["bias"][b] = of["n"].t().float() @ rows.float(), dbias
            grads["w_post"][b], grads["w_pre"][b] = dw_post, dw_pre
            dr, dn = new, rows @ self.w_in[b].to(self.dtype).t()
        first = torch.empty(w, device="cuda")
        self.norm.backward(kept[0]["r"], None, None, None, self.first, dr, dn, self._new(t, torch.float32), None, None, None,
                           first, ws)
        return [first, *grads["w_in"], *grads["bias"], *grads["w_post"], *grads["w_pre"]]

    def train_step(self, x, cu_seqlens, target, rate: float) -> torch.Tensor:
        """Gradient descent on the mean squared distance to `target`; the loss, on the device."""
        kept = []
        off = self.forward(x, cu_seqlens, kept=kept).float() - target
        for p, g in zip(self.parameters(), self.backward((2.0 * off / off.numel()).to(self.dtype), cu_seqlens, kept)):
            p -= rate * g
        return off.square().mean()


def _packed(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).cuda()


def train(width, blocks, tokens, steps, rate=0.5):
    """Losses of a student that learns a teacher's outputs."""
    cu = _packed([tokens // 2, tokens // 8, tokens - tokens // 2 - tokens // 8])
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(tokens, width, generator=gen, device="cuda")
    teacher, student = Stack(width, blocks, seed=1), Stack(width, blocks, seed=1)
    for w in student.w_in:
        w += 0.3 * torch.randn(w.shape, generator=gen, device="cuda") / width ** 0.5
    target = teacher.forward(x, cu).float()
    return [float(student.train_step(x, cu, target, rate)) for _ in range(steps)]


def serve(width, blocks, lengths, new):
    """Largest difference, over the rms, of prompts and single tokens from whole sequences."""
    stack = Stack(width, blocks)
    gen = torch.Generator(device="cuda").manual_seed(9)
    whole = [torch.randn(n + new, width, generator=gen, device="cuda") for n in lengths]
    want = stack.forward(torch.cat(whole), _packed([n + new for n in lengths])).split([n + new for n in lengths])
    states = torch.zeros(blocks, len(lengths) + 2, width, device="cuda")
    slots = torch.randperm(len(lengths) + 2, generator=gen, device="cuda")[:len(lengths)].to(torch.int32)
    got = [[y] for y in stack.forward(torch.cat([w[:n] for w, n in zip(whole, lengths)]), _packed(lengths), states, slots)
           .split(lengths)]
    for i in range(new):
        y = stack.token(torch.stack([w[n + i] for w, n in zip(whole, lengths)]), states, slots)
        for g, row in zip(got, y):
            g.append(row[None])
    off = torch.cat([torch.cat(g) - w for g, w in zip(got, want)]).float()
    return float(off.abs().max() / torch.cat(want).float().square().mean().sqrt())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    losses = train(a.width, a.blocks, a.tokens, a.steps)
    print("training: loss " + " ".join(f"{x:.4f}" for x in losses[::max(1, a.steps // 5)]) + f" ... {losses[-1]:.4f}")
    off = serve(a.width, a.blocks, [a.tokens // 2, 1, a.tokens // 3], 8)
    print(f"serving: prompts and single tokens differ from whole sequences by {off:.3g} of the rms at most")


if __name__ == "__main__":
    main()
