"""Plain 64-bit forms of the recurrent block's operators, token by token on the CPU, and how far a kernel
that computes in 32 bits may be from them.

U is half a step of f32.  `half` is half a step of a row type (torch.finfo(t).eps / 2), for the one rounding
of a result.  Bounds count roundings: a sum of n terms taken in any order is off by at most n U sum|terms|.
"""
import torch

U = 2.0 ** -24
GROUP = 32
SEGMENT = 128


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype):
    """Of a result: half a step relative, nothing for f32 results (their bounds hold it)."""
    return half(dtype) if dtype != torch.float32 else U


def d(t):
    return t.detach().cpu().double()


# ---- 8 bits --------------------------------------------------------------------------


def pack8(x):
    """Codes and scales of rows (any float type) by the definition."""
    x = d(x)
    tokens, width = x.shape
    groups = -(-width // GROUP)
    codes, scales = torch.zeros(tokens, width, dtype=torch.int8), torch.zeros(tokens, groups, dtype=torch.uint8)
    for k in range(groups):
        part = x[:, k * GROUP:(k + 1) * GROUP]
        most = part.abs().amax(1)
        finite = torch.isfinite(part).all(1)
        e = torch.full_like(most, -127)
        for _ in range(2 ** 8):  # the least power of two that holds the group
            e = torch.where(finite & (most > 127 * torch.exp2(e)), e + 1, e)
        codes[:, k * GROUP:(k + 1) * GROUP] = torch.where(
            finite[:, None], torch.round(torch.where(finite[:, None], part, 0.0) / torch.exp2(e)[:, None]), 0.0).to(torch.int8)
        scales[:, k] = torch.where(finite, e + 127, 255.0).to(torch.uint8)
    return codes, scales


def unpack8(codes, scales):
    codes, scales = d(codes), scales.cpu()
    step = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return codes * step.repeat_interleave(GROUP, 1)[:, :codes.shape[1]]


# ---- the recurrence ------------------------------------------------------------------


def recurrence(x, f, bias, lengths, state, complement):
    """h, the states before every token, the states left, a.  Rows of no sequence: NaN."""
    g = f + (0 if bias is None else bias)
    a, z = torch.sigmoid(g), torch.sigmoid(-g)
    h, before = torch.full_like(x, torch.nan), torch.full_like(x, torch.nan)
    left, row = state.clone(), 0
    for n, length in enumerate(lengths):
        now = state[n]
        for t in range(row, row + length):
            before[t] = now
            now = a[t] * now + (z[t] * x[t] if complement else x[t])
            h[t] = now
        left[n], row = now, row + length
    return h, before, left, a, z


def recurrence_grad(x, a, z, before, lengths, dh, dstate, complement):
    """dx, df, dbias, dstate_in, G."""
    dx, df, G = torch.full_like(x, torch.nan), torch.full_like(x, torch.nan), torch.full_like(x, torch.nan)
    into, row = dstate.clone(), 0
    dbias = torch.zeros(x.shape[1], dtype=x.dtype)
    for n, length in enumerate(lengths):
        now = dstate[n]
        for t in range(row + length - 1, row - 1, -1):
            now = dh[t] + now
            G[t] = now
            dx[t] = z[t] * now if complement else now
            df[t] = now * a[t] * z[t] * (before[t] - x[t] if complement else before[t])
            dbias += df[t]
            now = a[t] * now
        into[n], row = now, row + length
    return dx, df, dbias, into, G


def chain_bound(z, f, size):
    """How far a chain's values may be off, for each channel [1, channels]: `size` bounds what is added and
    the values themselves.  A token rounds its value a few times (4 U size, also where maps of segments are
    joined instead), and its gate is off by (|f| + 8) U relative to the smaller of a and 1 - a (exp of f: the
    product with log2 e is off by |f| U; a sum, a quotient); what has been lost decays with a, so at most
    1 / (1 - a) tokens count."""
    if not z.shape[0]:
        return U * size
    memory = torch.minimum(1 / z.amin(0).clamp(min=1e-30), torch.tensor(float(z.shape[0])))
    return U * (8 * memory + 4 * f.abs().amax(0) + 40) * size


# ---- the norms -----------------------------------------------------------------------


def act(kind, g):
    """The gate's factor and its slope."""
    if kind is None:
        return None, None
    p = torch.sigmoid(g)
    q = torch.sigmoid(-g)
    return {"linear": (g, torch.ones_like(g)), "sigmoid": (p, p * q), "silu": (g * p, p + g * p * q)}[kind]


def rms(x, eps):
    return (x.square().mean(-1, keepdim=True) + eps).sqrt()
