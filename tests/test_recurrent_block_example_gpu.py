"""The recurrent block's operators as a program runs them together: examples/recurrent_block.py."""
import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "recurrent_block.py"
    spec = importlib.util.spec_from_file_location("recurrent_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_training_runs():
    losses = _example().train(128, 2, 512, 3)
    assert len(losses) == 3 and all(x == x and x < float("inf") for x in losses)


def test_serving_agrees_with_whole_sequences():
    # bf16 rows between the operators: a state that differs in its last f32 digits may round h the other way,
    # one step of bf16 of a value up to about 4 rms (2^-7 * 4), through two blocks
    assert _example().serve(128, 2, [300, 1, 140], 4) <= 2 * 2.0 ** -7 * 4


def _plain(stack, x, lengths):
    """The stack from elementary operations in 64 bits, on leaves that autograd follows."""
    leaves = [p.detach().cpu().double().requires_grad_() for p in stack.parameters()]
    n = stack.blocks
    first, w_in, bias = leaves[0], leaves[1:1 + n], leaves[1 + n:1 + 2 * n]
    w_post, w_pre = leaves[1 + 2 * n:1 + 3 * n], leaves[1 + 3 * n:]
    norm = lambda v, w: w * v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    r = x.cpu().double()
    y = norm(r, first)
    for b in range(n):
        v, f, g = (y @ w_in[b]).split(stack.width, 1)
        a, z = torch.sigmoid(f + bias[b]), torch.sigmoid(-(f + bias[b]))
        rows, at = [], 0
        for length in lengths:
            h = torch.zeros(stack.width, dtype=torch.float64)
            for t in range(at, at + length):
                h = a[t] * h + z[t] * v[t]
                rows.append(h)
            at += length
        r = r + 0.5 * norm(torch.stack(rows), w_post[b]) * g * torch.sigmoid(g)
        y = norm(r, w_pre[b])
    return y, leaves


def test_gradients_of_the_stack():
    """Outputs and gradients of every parameter against autograd's of the 64-bit form.

    In f32 rows the outputs are f32's; the activations that the gradients are made of are off by 1/127 of a group's
    largest value at most (8 bits), which is about 3 of its rms: a gradient's relative error stays below a few times
    3 / 127 / sqrt(3) = 1.4% a kept activation (uniform roundings), of which three enter each of the two blocks."""
    m = _example()
    lengths = [150, 37]
    stack = m.Stack(64, 2, dtype=torch.float32, seed=3)
    gen = torch.Generator("cuda").manual_seed(4)
    x, dy = torch.randn(187, 64, generator=gen, device="cuda"), torch.randn(187, 64, generator=gen, device="cuda")
    kept = []
    cu = torch.tensor([0, 150, 187], dtype=torch.int32, device="cuda")
    y = stack.forward(x, cu, kept=kept)
    want, leaves = _plain(stack, x, lengths)
    # (products in f32, TF32 off: 64 sums of 2^-24 each, through two blocks)
    assert float((y.cpu().double() - want.detach()).norm() / want.detach().norm()) < 1e-4
    (want * dy.cpu().double()).sum().backward()
    for got, leaf in zip(stack.backward(dy, cu, kept), leaves):
        off = float((got.cpu().double() - leaf.grad).norm() / leaf.grad.norm())
        assert off < 6 * 0.014, off
