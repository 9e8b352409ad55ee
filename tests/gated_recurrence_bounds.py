"""How far the gated recurrence's results may be from the 64-bit form, token by token.

Errors run through the recurrences themselves: what a token adds is kept by the tokens behind it as its value is.
U is half a step of f32.  What a token adds, with m the smaller of a and 1 - a and g = f + bias:

* its gate: m is off by gate(g) = (3 |g| + 8) U relative to itself (the sum and the product with log2 e, |g| U each,
  log2 e itself; 2^t: 2^-22; a sum, a reciprocal of 2^-23, a product), the larger one by no more than that and U;
* its roundings: of the difference or sum that m multiplies, of the step, of the product of gates (`STEP` = 3).

A chain of 16 tokens starts from zero, what enters it is added with the product of its gates; so the values that are
rounded are at most the true one and what entered the chain.  Chains are joined to segments of 128 tokens (a product and
a sum a chain: 2 U), segments to sequences (the same).  Gradients: what leaves a chain is a sum of 16 products with up to 16
roundings each (32 U of the sum of their sizes).
"""
import torch

from tests.recurrent_block_oracle import U

CHAIN, SEGMENT, STEP = 16, 128, 3


def gate(g):
    return (3 * g.abs() + 8) * U


def values(x, g, a, z, h, before, lengths, entered, complement, heads=None):
    """Bounds on h after every token, and before it, [tokens, channels].

    entered: the states that enter the sequences; `heads`: bounds on them (0 where they are given)."""
    after, ahead = torch.zeros_like(x), torch.zeros_like(x)
    small, off = torch.minimum(a, z), gate(g)
    row = 0
    for n, length in enumerate(lengths):
        err = torch.zeros_like(x[0]) if heads is None else heads[n].clone()
        for i in range(length):
            t = row + i
            if i % CHAIN == 0:
                chain = before[t].abs()
            if i % SEGMENT == 0:
                segment = before[t].abs()
            ahead[t] = err
            size = before[t].abs() + chain + x[t].abs()  # of what the gate multiplies, at most
            err = a[t] * err + off[t] * small[t] * size + U * (small[t] * size if complement else size) + \
                (STEP - 1) * U * (h[t].abs() + chain)
            if i % CHAIN == CHAIN - 1:
                err = err + 2 * U * (h[t].abs() + chain + segment)
            if i % SEGMENT == SEGMENT - 1:
                err = err + 2 * U * (h[t].abs() + segment)
            after[t] = err + U * (h[t].abs() + chain)  # (the output's own sum)
        row += length
    return after, ahead


def gradients(g, a, z, G, dh, dstate, lengths):
    """Bounds on G of every token and on the gradients of the entering states."""
    of_g, into = torch.zeros_like(dh), torch.zeros_like(dstate)
    small, off = torch.minimum(a, z), gate(g)
    row = 0
    for n, length in enumerate(lengths):
        err = torch.zeros_like(dstate[0])
        for i in range(length - 1, -1, -1):
            t = row + i
            if i == length - 1 or i % CHAIN == CHAIN - 1:
                behind, parts = (dstate[n] if i == length - 1 else a[t + 1] * G[t + 1]).abs(), torch.zeros_like(err)
            if i == length - 1 or i % SEGMENT == SEGMENT - 1:
                segment = behind
            of_g[t] = err + U * (G[t].abs() + behind)
            parts = a[t] * (dh[t].abs() + parts)
            left = (a[t] * G[t]).abs()
            err = a[t] * of_g[t] + off[t] * small[t] * (G[t].abs() + behind) + STEP * U * (left + a[t] * behind)
            if i % CHAIN == 0:
                err = err + 32 * U * parts + 2 * U * (left + behind + segment)
            if i % SEGMENT == 0:
                err = err + 2 * U * (left + segment)
        into[n], row = err, row + length
    return of_g, into
