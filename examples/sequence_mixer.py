#!/usr/bin/env python
"""A mixer layer of a decayed linear-attention model on the sequence operators.

    python examples/sequence_mixer.py [--width 512] [--heads 8] [--kv-heads 4] [--tokens 1024] [--steps 20]

One layer: a projection to packed query / key / value rows, the norm of every
query and key head with the rotation by position (QkNormRotary), linear attention
with a decay for each head (LinearAttention), and a projection back.

* Training: packed sequences of different lengths, the operators' own backward
  passes, plain gradient descent on the distance to a teacher layer's outputs.
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


class Mixer:
    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int = 64, dtype=torch.bfloat16, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv, self.dim, self.dtype = heads, kv_heads, head_dim, dtype
        rows = (heads + 2 * kv_heads) * head_dim
        self.w_in = torch.randn(width, rows, generator=gen, device="cuda") / width ** 0.5
        self.w_out = torch.randn(heads * head_dim, width, generator=gen, device="cuda") / (heads * head_dim) ** 0.5
        self.wq, self.wk = torch.ones(head_dim, device="cuda"), torch.ones(head_dim, device="cuda")
        self.log_decay = -2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)
        self.qk = sequence.QkNormRotary(dtype, heads, kv_heads, head_dim)
        self.attention = sequence.LinearAttention(dtype, heads, kv_heads, head_dim, head_dim)

    def _rows(self, x):
        """Packed rows of a projection and their query, key and value heads (views)."""
        rows = x.to(self.dtype) @ self.w_in.to(self.dtype)
        h, k, d = self.heads, self.kv, self.dim
        t = rows.shape[0]
        return rows, rows[:, :h * d].view(t, h, d), rows[:, h * d:(h + k) * d].view(t, k, d), \
            rows[:, (h + k) * d:].view(t, k, d)

    def _mix_in(self, x, positions):
        _, q, k, v = self._rows(x)
        qn, kn = torch.empty(q.shape, dtype=q.dtype, device="cuda"), torch.empty(k.shape, dtype=k.dtype, device="cuda")
        self.qk.forward(q, k, positions, self.wq, self.wk, qn, kn, stream=_stream())
        return q, k, v, qn, kn

    def prompt(self, x, positions, cu_seqlens, state=None, slots=None):
        """Outputs of packed sequences; their states are continued from and left in `state`."""
        _, _, v, qn, kn = self._mix_in(x, positions)
        o = torch.empty_like(qn)
        ws = torch.empty(self.attention.workspace_bytes(x.shape[0], cu_seqlens.numel() - 1), dtype=torch.uint8,
                         device="cuda")
        self.attention.forward(qn, kn, v, self.log_decay, cu_seqlens, o, state_in=state, state_out=state, slots=slots,
                               workspace=ws, stream=_stream())
        return o.flatten(1).float() @ self.w_out

    def token(self, x, positions, state, slots=None):
        """One token of each request."""
        _, _, v, qn, kn = self._mix_in(x, positions)
        o = torch.empty_like(qn)
        self.attention.step(qn, kn, v, self.log_decay, state, o, slots=slots, stream=_stream())
        return o.flatten(1).float() @ self.w_out

    def train_step(self, x, positions, cu_seqlens, target, rate: float) -> torch.Tensor:
        """Gradient descent on the mean squared distance to `target`; the loss, on the device."""
        t, n = x.shape[0], cu_seqlens.numel() - 1
        q, k, v, qn, kn = self._mix_in(x, positions)
        o = torch.empty_like(qn)
        ws = torch.empty(max(self.attention.workspace_bytes(t, n), self.attention.backward_workspace_bytes(t, n),
                             self.qk.workspace_bytes(t)), dtype=torch.uint8, device="cuda")
        self.attention.forward(qn, kn, v, self.log_decay, cu_seqlens, o, workspace=ws, stream=_stream())
        flat = o.flatten(1).float()
        off = flat @ self.w_out - target
        dy = 2.0 * off / off.numel()
        do = (dy @ self.w_out.t()).to(self.dtype).view_as(o)
        dqn, dkn = torch.empty_like(qn), torch.empty_like(kn)
        rows = torch.empty(t, self.w_in.shape[1], dtype=self.dtype, device="cuda")  # gradients of the packed rows
        h, g, d = self.heads, self.kv, self.dim
        dq, dk, dv = rows[:, :h * d].view(t, h, d), rows[:, h * d:(h + g) * d].view(t, g, d), \
            rows[:, (h + g) * d:].view(t, g, d)
        self.attention.backward(qn, kn, v, self.log_decay, cu_seqlens, do, dqn, dkn, dv, workspace=ws, stream=_stream())
        dwq, dwk = torch.empty_like(self.wq), torch.empty_like(self.wk)
        self.qk.backward(q, k, positions, self.wq, self.wk, dqn, dkn, dq, dk, dwq, dwk, ws, stream=_stream())
        self.w_out -= rate * (flat.t() @ dy)
        self.w_in -= rate * (x.t() @ rows.float())
        self.wq -= rate * dwq
        self.wk -= rate * dwk
        return off.square().mean()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _packed(lengths):
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    positions = torch.cat([torch.arange(n) for n in lengths]).to(torch.int32).view(1, -1).cuda()
    return cu, positions


def train(width, heads, kv_heads, tokens, steps, rate=0.03):
    """Losses of a student layer that learns a teacher's outputs."""
    lengths = [tokens // 2, tokens // 8, tokens - tokens // 2 - tokens // 8]
    cu, positions = _packed(lengths)
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(tokens, width, generator=gen, device="cuda")
    teacher, student = Mixer(width, heads, kv_heads, seed=1), Mixer(width, heads, kv_heads, seed=1)
    student.w_in += 0.3 * torch.randn(student.w_in.shape, generator=gen, device="cuda") / width ** 0.5
    student.w_out += 0.3 * torch.randn(student.w_out.shape, generator=gen, device="cuda") / student.w_out.shape[0] ** 0.5
    target = teacher.prompt(x, positions, cu)
    return [float(student.train_step(x, positions, cu, target, rate)) for _ in range(steps)]


def serve(width, heads, kv_heads, lengths, new):
    """Largest difference, over the rms, of prompts and single tokens from whole sequences."""
    mixer = Mixer(width, heads, kv_heads)
    gen = torch.Generator(device="cuda").manual_seed(9)
    whole = [torch.randn(n + new, width, generator=gen, device="cuda") for n in lengths]
    cu, positions = _packed([n + new for n in lengths])
    want = mixer.prompt(torch.cat(whole), positions, cu).split([n + new for n in lengths])
    state = torch.zeros(len(lengths) + 2, heads, mixer.dim, mixer.dim, device="cuda")
    slots = torch.randperm(len(lengths) + 2, generator=gen, device="cuda")[:len(lengths)].to(torch.int32)
    cu, positions = _packed(lengths)
    got = [[y] for y in mixer.prompt(torch.cat([w[:n] for w, n in zip(whole, lengths)]), positions, cu, state,
                                     slots).split(lengths)]
    for i in range(new):
        at = torch.tensor([[n + i for n in lengths]], dtype=torch.int32, device="cuda")
        y = mixer.token(torch.stack([w[n + i] for w, n in zip(whole, lengths)]), at, state, slots)
        for g, row in zip(got, y):
            g.append(row[None])
    off = torch.cat([torch.cat(g) - w for g, w in zip(got, want)])
    return float(off.abs().max() / torch.cat(want).square().mean().sqrt())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--width", type=int, default=512)
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    losses = train(a.width, a.heads, a.kv_heads, a.tokens, a.steps)
    print("training: loss " + " ".join(f"{x:.4f}" for x in losses[::max(1, a.steps // 5)]) + f" ... {losses[-1]:.4f}")
    off = serve(a.width, a.heads, a.kv_heads, [a.tokens // 2, 1, a.tokens // 3], 8)
    print(f"serving: prompts and single tokens differ from whole sequences by {off:.3g} of the rms at most")


if __name__ == "__main__":
    main()
