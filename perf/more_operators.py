"""Cases of a recurrent block's operators: the gated linear recurrence, the norms around a block with its
gate and residual scale, and activations kept in 8 bits for the backward pass.

`own` false computes each operator from elementary torch operations in 32 bits,
`own` true calls `tensoroperations_b200.sequence`.  `exact` computes the same
outputs from the definitions (token by token) in 64 bits.
"""
import functools
import math
import random

import torch

own = False

DEVICE = "cuda"
GROUP = 32  # values that share a scale in 8 bits
SEGMENT = 128  # tokens between the states that the recurrence's forward pass saves for its gradients


def listed():
    return [
        # one new token of a few running requests: the call's own latency counts
        dict(name="step 5 requests", op="step", requests=5, channels=1024, complement=True, dtype="bf16"),
        # decoding a full batch: the states are the traffic
        dict(name="step 512 requests", op="step", requests=512, channels=8192, complement=True, dtype="bf16"),
        # prompts of many requests packed together, continued from and written to their state slots
        dict(name="prompts packed", op="prompt", tokens=9001, seqs=11, channels=2560, complement=True, states=True,
             dtype="bf16"),
        # one long document: the time axis has to be split
        dict(name="prompt long", op="prompt", tokens=49152, seqs=1, channels=4096, complement=True, states=False,
             dtype="bf16"),
        # a training step of the recurrence on equal sequences, its inputs kept in 8 bits
        dict(name="training 8-bit", op="train", tokens=16384, seqs=4, channels=4096, complement=True, states=False,
             keep=True, dtype="bf16"),
        # a training step on ragged sequences with gradients of the states, odd width, inputs as they are
        dict(name="training ragged", op="train", tokens=1501, seqs=5, channels=333, complement=False, states=True,
             keep=False, dtype="f32"),
        # between two blocks, one new token of 24 requests
        dict(name="norms 24 tokens", op="norm", tokens=24, width=2048, gate="silu", dtype="bf16", residual="bf16"),
        # between two blocks, a training batch whose residual stream is held in 32 bits
        dict(name="norms batch", op="norm", tokens=16384, width=4096, gate="silu", dtype="bf16", residual="f32"),
        # their gradients, from activations kept in 8 bits
        dict(name="norm gradients 8-bit", op="norm_grad", tokens=8192, width=4096, gate="silu", keep=True, dtype="bf16",
             residual="bf16"),
        # gradients without a gate at an odd width, from the activations themselves
        dict(name="norm gradients odd", op="norm_grad", tokens=6137, width=1003, gate="none", keep=False, dtype="f32",
             residual="f32"),
        # a batch's activations into 8 bits and back
        dict(name="8 bits batch", op="store", tokens=16384, width=4096, dtype="bf16"),
        # the same at an odd width, in the framework's own type
        dict(name="8 bits odd", op="store", tokens=777, width=1237, dtype="f32"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["step", "prompt", "prompt", "train", "train", "norm", "norm_grad", "norm_grad", "store"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    width = rng.choice([_log_uniform(rng, 33, 8192), 64 * _log_uniform(rng, 1, 128)])
    if op in ("norm", "norm_grad", "store"):
        most = {"norm": 16384, "norm_grad": 8192, "store": 16384}[op] * 4096 // (width * (2 if dtype == "f32" else 1))
        case = dict(op=op, tokens=_log_uniform(rng, 1, min(most, 65536)), width=width, dtype=dtype)
        if op == "store":
            return case
        case.update(gate=rng.choice(["none", "silu", "sigmoid", "linear"]),
                    residual="f32" if dtype == "f32" else rng.choice(["bf16", "f32"]))
        return dict(case, keep=rng.random() < 0.5) if op == "norm_grad" else case
    base = dict(op=op, channels=width, complement=rng.random() < 0.7, dtype=dtype)
    if op == "step":
        return dict(base, requests=_log_uniform(rng, 1, min(512, 512 * 8192 // width)))
    most = (49152 if op == "prompt" else 16384) * 4096 // (width * (2 if dtype == "f32" else 1))
    tokens = _log_uniform(rng, 1, min(most, 49152 if op == "prompt" else 16384))
    case = dict(base, tokens=tokens, seqs=min(tokens, _log_uniform(rng, 1, 32)), states=rng.random() < 0.5)
    return dict(case, keep=rng.random() < 0.5) if op == "train" else case


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _lengths(case):
    """Ragged lengths with the case's total; equal ones for a training batch without states."""
    n, total = case["seqs"], case["tokens"]
    if case["op"] == "train" and not case["states"] and total % n == 0:
        return [total // n] * n
    cut = random.Random(total * 131 + n)
    cuts = sorted(cut.randint(0, total) for _ in range(n - 1))
    if n >= 4:
        cuts[1] = cuts[0]  # an empty sequence among them
    if n >= 5:
        cuts[3] = max(cuts[2], min(cuts[2] + 1, total))  # and one of a single token
        cuts.sort()
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _type(case["dtype"])

    def normal(*shape, t=None):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(t or dtype)

    s = dict(case=case)
    if case["op"] == "store":  # activations: a few channels are far larger than the others
        loud = torch.exp(1.5 * normal(case["width"], t=torch.float32))
        s["x"] = (normal(case["tokens"], case["width"], t=torch.float32) * loud).to(dtype)
        return s
    if case["op"] in ("norm", "norm_grad"):
        T, w = case["tokens"], case["width"]
        residual = _type(case["residual"])
        s["r"] = 2 * normal(T, w, t=residual)  # norm_grad: the stream after the block
        s["y"] = normal(T, w)
        if case["gate"] != "none":
            s["g"] = normal(T, w)
        s["w_post"] = 1 + 0.2 * normal(w, t=torch.float32)
        s["w_pre"] = 1 + 0.2 * normal(w, t=torch.float32)
        if case["op"] == "norm_grad":
            s["dn"], s["dr"] = normal(T, w), normal(T, w, t=residual)
            if case["keep"]:  # what is left of the forward pass: codes and scales
                for n in ("r", "y", "g"):
                    if n in s:
                        s[n] = _pack(s[n].to(torch.float32))
        return s
    T, c = case["requests"] if case["op"] == "step" else case["tokens"], case["channels"]
    rows = normal(T, 2 * c)  # a projection's packed rows: values, gates
    s["x"], s["f"] = rows[:, :c], rows[:, c:]
    # biases that spread the channels' memory from a few tokens to thousands
    s["bias"] = 1 + 7 * torch.rand(c, generator=gen, device=DEVICE)
    if case["op"] == "step":
        s["state"] = normal(T + 3, c, t=torch.float32)
        s["slots"] = torch.randperm(T + 3, generator=gen, device=DEVICE)[:T].to(torch.int32)
        return s
    n = case["seqs"]
    s["lengths"] = _lengths(case)
    s["cu_seqlens"] = torch.tensor([0] + s["lengths"]).cumsum(0).to(torch.int32).to(DEVICE)
    if case["states"]:
        s["state"] = normal(n + 2, c, t=torch.float32)
        s["slots"] = torch.randperm(n + 2, generator=gen, device=DEVICE)[:n].to(torch.int32)
    if case["op"] == "train":
        s["dh"] = normal(T, c)
        if case["states"]:
            s["dstate"] = normal(n, c, t=torch.float32)
    return s


# ---- the framework's operators ---------------------------------------------------


@functools.lru_cache(maxsize=None)
def _operator(op, dtype, width, *more):
    from tensoroperations_b200 import sequence
    if op == "recurrence":
        return sequence.GatedRecurrence(dtype, width, complement=more[0])
    if op == "norm":
        return sequence.BlockNorm(dtype, width, residual=more[0], gate=None if more[1] == "none" else more[1], scale=0.5)
    return sequence.Checkpoint8(dtype, width)


def _run_own(s):
    case = s["case"]
    new = functools.partial(torch.empty, device=DEVICE)
    if case["op"] == "store":
        from tensoroperations_b200 import sequence
        op = _operator("store", case["dtype"], case["width"])
        x8 = sequence.Rows8.empty(case["tokens"], case["width"], DEVICE)
        op.pack(s["x"], x8)
        x = torch.empty_like(s["x"])
        op.unpack(x8, x)
        return x
    if case["op"] in ("norm", "norm_grad"):
        op = _operator("norm", case["dtype"], case["width"], case["residual"], case["gate"])
        if case["op"] == "norm":
            r, n = torch.empty_like(s["r"]), torch.empty_like(s["y"])
            op.forward(s["r"], s["y"], s.get("g"), s["w_post"], s["w_pre"], r, n)
            return dict(r=r, n=n)
        r, y, g = (s.get(n) for n in ("r", "y", "g"))
        if case["keep"]:
            from tensoroperations_b200 import sequence
            r, y, g = (x if x is None else sequence.Rows8(*x) for x in (r, y, g))
        dr, dy = torch.empty_like(s["dr"]), torch.empty_like(s["dn"])
        dg = None if g is None else torch.empty_like(s["dn"])
        dw_post, dw_pre = torch.empty_like(s["w_post"]), torch.empty_like(s["w_pre"])
        ws = new(op.workspace_bytes(case["tokens"]), dtype=torch.uint8)
        op.backward(r, y, g, s["w_post"], s["w_pre"], s["dr"], s["dn"], dr, dy, dg, dw_post, dw_pre, ws)
        out = dict(dr=dr, dy=dy, dw_post=dw_post, dw_pre=dw_pre)
        return out if g is None else dict(out, dg=dg)
    c = case["channels"]
    op = _operator("recurrence", case["dtype"], c, case["complement"])
    x, f, bias = s["x"], s["f"], s["bias"]
    h = new(x.shape[0], c, dtype=x.dtype)
    if case["op"] == "step":
        op.step(x, f, bias, s["state"], h, slots=s["slots"])
        return dict(h=h, state=s["state"])
    T, n, cu = case["tokens"], case["seqs"], s["cu_seqlens"]
    ws = new(op.workspace_bytes(T, n), dtype=torch.uint8)
    if case["op"] == "prompt":
        if case["states"]:
            op.forward(x, f, bias, cu, h, state_in=s["state"], state_out=s["state"], slots=s["slots"], workspace=ws)
            return dict(h=h, state=s["state"])
        state = new(n, c)
        op.forward(x, f, bias, cu, h, state_out=state, workspace=ws)
        return dict(h=h, state=state)
    saved = new(op.saved_rows(T, n), c)
    kept = dict()
    if case["keep"]:
        from tensoroperations_b200 import sequence
        kept = dict(keep_x=sequence.Rows8.empty(T, c, DEVICE), keep_f=sequence.Rows8.empty(T, c, DEVICE))
    states = dict(state_in=s["state"], slots=s["slots"]) if case["states"] else {}
    op.forward(x, f, bias, cu, h, saved=saved, workspace=ws, **states, **kept)
    dx, df, dbias = new(T, c, dtype=x.dtype), new(T, c, dtype=x.dtype), new(c)
    ws = new(op.backward_workspace_bytes(T, n), dtype=torch.uint8)
    dstate = new(n, c) if case["states"] else None
    op.backward(kept.get("keep_x", x), kept.get("keep_f", f), bias, cu, saved, s["dh"], dx, df, dbias,
                dstate_out=s.get("dstate"), dstate_in=dstate, workspace=ws)
    out = dict(h=h, dx=dx, df=df, dbias=dbias)
    return dict(out, dstate=dstate) if case["states"] else out


# ---- plain forms -----------------------------------------------------------------


def _pack(x):
    """Codes and scales of rows in 8 bits: groups of 32, scale 2^(byte-127), the least that holds the group."""
    tokens, width = x.shape
    pad = -width % GROUP
    groups = torch.nn.functional.pad(x, (0, pad)).view(tokens, -1, GROUP)
    m, k = torch.frexp(groups.abs().amax(-1))  # amax = m 2^k, 1/2 <= m < 1
    e = torch.where(m > 127 / 128, k - 6, k - 7)
    e = torch.where(m == 0, -127, e)
    codes = torch.ldexp(groups, -e[..., None].clamp(min=-126)).round()
    return codes.to(torch.int8).view(tokens, -1)[:, :width].contiguous(), (e + 127).to(torch.uint8)


def _unpack(packed):
    codes, scales = packed
    width = codes.shape[1]
    scale = torch.ldexp(torch.ones((), device=codes.device), scales.to(torch.int32) - 127)
    return codes.to(torch.float32) * scale.repeat_interleave(GROUP, 1)[:, :width]


def _act(g, gate):
    """The gate's factor and its slope."""
    if gate == "linear":
        return g, torch.ones_like(g)
    p = torch.sigmoid(g)
    if gate == "sigmoid":
        return p, p * (1 - p)
    return g * p, p * (1 + g * (1 - p))


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t over the first axis (h before the first token: 0), by doubling."""
    a, b = a.clone(), b.clone()
    step = 1
    while step < a.shape[0]:
        b[step:] += a[step:] * b[:-step].clone()
        a[step:] *= a[:-step].clone()
        step *= 2
    return b


def _segments(lengths):
    """Lengths of the pieces of SEGMENT tokens (the last one shorter) of the sequences that have tokens."""
    return [min(SEGMENT, n - i) for n in lengths for i in range(0, n, SEGMENT)]


def _ends(lengths):
    """First and last row of the sequences that have tokens, and which these are."""
    n = torch.tensor(lengths, device=DEVICE)
    last = n.cumsum(0) - 1
    at = (n > 0).nonzero()[:, 0]
    return (last - n + 1)[at], last[at], at


def _recur(x, f, bias, complement, lengths, state):
    """Outputs, the states left, and what the gradients use again."""
    z, a = torch.sigmoid(-(f + bias)), torch.sigmoid(f + bias)
    b = z * x if complement else x.clone()
    first, last, at = _ends(lengths)
    if len(at):
        b[first] += a[first] * state[at]
    cut = a.clone()
    cut[first] = 0
    h = _scan(cut, b)
    left = state.clone()
    left[at] = h[last]
    before = torch.cat((torch.zeros_like(h[:1]), h[:-1]))
    before[first] = state[at]
    return h, left, a, z, before


def _run_plain(s):
    case = s["case"]
    f32 = lambda t: t.to(torch.float32)  # noqa: E731
    dtype = _type(case["dtype"])
    if case["op"] == "store":
        return _unpack(_pack(f32(s["x"]))).to(dtype)
    if case["op"] in ("norm", "norm_grad"):
        residual = _type(case["residual"])
        r, y = ((_unpack(s[n]) if isinstance(s[n], tuple) else f32(s[n])) for n in ("r", "y"))
        post = ((y * y).mean(-1, keepdim=True) + 1e-6).rsqrt()
        u = y * post * s["w_post"]
        if case["gate"] != "none":
            g = _unpack(s["g"]) if isinstance(s["g"], tuple) else f32(s["g"])
            factor, slope = _act(g, case["gate"])
        if case["op"] == "norm":
            r = r + 0.5 * (u if case["gate"] == "none" else u * factor)
            n = r * ((r * r).mean(-1, keepdim=True) + 1e-6).rsqrt() * s["w_pre"]
            return dict(r=r.to(residual), n=n.to(dtype))
        pre = ((r * r).mean(-1, keepdim=True) + 1e-6).rsqrt()
        dn, hat = f32(s["dn"]), r * pre
        e = dn * s["w_pre"]
        t = f32(s["dr"]) + pre * (e - hat * (e * hat).mean(-1, keepdim=True))
        du = 0.5 * t
        out = dict(dr=t.to(residual), dw_pre=(dn * hat).sum(0))
        if case["gate"] != "none":
            out["dg"] = (du * u * slope).to(dtype)
            du = du * factor
        e, hat = du * s["w_post"], y * post
        return dict(out, dy=(post * (e - hat * (e * hat).mean(-1, keepdim=True))).to(dtype), dw_post=(du * hat).sum(0))
    x, f, bias = f32(s["x"]), f32(s["f"]), s["bias"]
    if case["op"] == "step":
        at = s["slots"].long()
        a = torch.sigmoid(f + bias)
        h = a * s["state"][at] + (torch.sigmoid(-(f + bias)) * x if case["complement"] else x)
        s["state"][at] = h
        return dict(h=h.to(dtype), state=s["state"])
    n, lengths = case["seqs"], s["lengths"]
    state = s["state"][s["slots"].long()] if case["states"] else torch.zeros(n, case["channels"], device=DEVICE)
    h, left, a, z, before = _recur(x, f, bias, case["complement"], lengths, state)
    if case["op"] == "prompt":
        if case["states"]:
            s["state"][s["slots"].long()] = left
            left = s["state"]
        return dict(h=h.to(dtype), state=left)
    if case["keep"]:  # the gradients are those of the values kept, from the states that the forward pass saved
        x, f = _unpack(_pack(x)), _unpack(_pack(f))
        pieces = _segments(lengths)
        _, _, a, z, before = _recur(x, f, bias, case["complement"], pieces, before[_ends(pieces)[0]])
    first, last, at = _ends(lengths)
    b = f32(s["dh"])
    if case["states"]:
        b = b.clone()
        b[last] += s["dstate"][at]
    later = torch.cat((a[1:], torch.zeros_like(a[:1])))  # a of the next token
    later[last] = 0
    G = _scan(later.flip(0), b.flip(0)).flip(0)
    df = G * a * z * (before - x if case["complement"] else before)
    out = dict(h=h.to(dtype), dx=(z * G if case["complement"] else G).to(dtype), df=df.to(dtype),
               dbias=df.sum(0, dtype=torch.float64).to(torch.float32))
    if case["states"]:
        out["dstate"] = s["dstate"].clone()
        out["dstate"][at] = a[first] * G[first]
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "store":  # read, kept, read again, written
        values = case["tokens"] * case["width"]
        return dict(bytes=values * 2 * (size + 1 + 1 / GROUP), flops=4 * values)
    if case["op"] in ("norm", "norm_grad"):
        values, r = case["tokens"] * case["width"], 2 if case["residual"] == "bf16" else 4
        gate = case["gate"] != "none"
        if case["op"] == "norm":
            return dict(bytes=values * (2 * r + (2 + gate) * size) + 8 * case["width"], flops=(10 + 6 * gate) * values)
        kept = (2 + gate) * (1 + 1 / GROUP) if case["keep"] else r + (1 + gate) * size
        return dict(bytes=values * (kept + 2 * r + (2 + gate) * size) + 16 * case["width"],
                    flops=(26 + 10 * gate) * values)
    c = case["channels"]
    if case["op"] == "step":
        return dict(bytes=case["requests"] * c * (3 * size + 8), flops=10 * case["requests"] * c)
    values, states = case["tokens"] * c, case["seqs"] * c * 4
    if case["op"] == "prompt":
        return dict(bytes=3 * values * size + states * (2 if case["states"] else 1), flops=10 * values)
    # x, f read and h written; both kept in 8 bits, or read again; dh read, dx and df written
    kept = 4 * (1 + 1 / GROUP) if case["keep"] else 2 * size
    return dict(bytes=values * (6 * size + kept) + (3 * states if case["states"] else 0) + 8 * c, flops=40 * values)


# ---- the definitions, token by token, in 64 bits -------------------------------------


def _kept(x):
    """The values that rows in 8 bits stand for."""
    out = torch.zeros_like(x)
    for part, to in zip(x.split(GROUP, 1), out.split(GROUP, 1)):
        most = part.abs().amax(1, keepdim=True)
        # (log2 of 127 2^k may come out above k; the next value of 24 bits lies 1e-7 higher)
        step = torch.exp2(torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / 127) - 1e-9))
        to.copy_(torch.round(part / step) * step)
    return out


def _walk(lengths):
    """For each time step, the sequences that have such a token (longest first), and its packed row."""
    first = [sum(lengths[:n]) for n in range(len(lengths))]
    length, first = torch.tensor(lengths, device=DEVICE), torch.tensor(first, device=DEVICE)
    order = torch.argsort(length, descending=True, stable=True)
    ordered, first = sorted(lengths, reverse=True), first[order]
    live = len(lengths)
    for t in range(max(lengths, default=0)):
        while live and ordered[live - 1] <= t:
            live -= 1
        yield order[:live], first[:live] + t


def _steps(x, f, bias, complement, lengths, state):
    """h after every token and before it, the states left, a of every token."""
    a = 1 / (1 + torch.exp(-(f + bias)))
    state = state.clone()
    h, before = torch.zeros_like(x), torch.zeros_like(x)
    for at, row in _walk(lengths):
        now = state[at]
        before[row] = now
        now = a[row] * now + ((1 - a[row]) * x[row] if complement else x[row])
        h[row] = now
        state[at] = now
    return h, before, state, a


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: t.to(torch.float64)  # noqa: E731
    if case["op"] == "store":
        return _kept(d(s["x"]))
    if case["op"] in ("norm", "norm_grad"):
        def value(t):
            if not isinstance(t, tuple):
                return d(t)
            step = torch.exp2(d(t[1]) - 127)
            return d(t[0]) * step[:, torch.arange(t[0].shape[1], device=DEVICE) // GROUP]

        r, y = value(s["r"]), value(s["y"])
        g = value(s["g"]) if case["gate"] != "none" else None
        logistic = None if g is None else 1 / (1 + torch.exp(-g))
        factor = {"none": lambda: torch.ones_like(y), "linear": lambda: g, "sigmoid": lambda: logistic,
                  "silu": lambda: g * logistic}[case["gate"]]()
        length = (y.square().sum(-1, keepdim=True) / case["width"] + 1e-6).sqrt()
        w_post, w_pre = d(s["w_post"]), d(s["w_pre"])
        if case["op"] == "norm":
            r = r + 0.5 * factor * w_post * y / length
            return dict(r=r, n=w_pre * r / (r.square().sum(-1, keepdim=True) / case["width"] + 1e-6).sqrt())
        size = (r.square().sum(-1, keepdim=True) / case["width"] + 1e-6).sqrt()
        dn, e = d(s["dn"]), d(s["dn"]) * w_pre
        t = d(s["dr"]) + e / size - r * (e * r).sum(-1, keepdim=True) / (case["width"] * size ** 3)
        e = 0.5 * t * factor * w_post
        out = dict(dr=t, dw_pre=(dn * r / size).sum(0), dw_post=(0.5 * t * factor * y / length).sum(0),
                   dy=e / length - y * (e * y).sum(-1, keepdim=True) / (case["width"] * length ** 3))
        if g is not None:
            slope = {"linear": lambda: 1.0, "sigmoid": lambda: logistic * (1 - logistic),
                     "silu": lambda: logistic + g * logistic * (1 - logistic)}[case["gate"]]()
            out["dg"] = 0.5 * t * slope * w_post * y / length
        return out
    x, f, bias = d(s["x"]), d(s["f"]), d(s["bias"])
    if case["op"] == "step":
        state = d(s["state"])
        for i, slot in enumerate(s["slots"].tolist()):
            a = 1 / (1 + torch.exp(-(f[i] + bias)))
            state[slot] = a * state[slot] + ((1 - a) * x[i] if case["complement"] else x[i])
        return dict(h=state[s["slots"].long()], state=state)
    n, lengths, comp = case["seqs"], s["lengths"], case["complement"]
    state = d(s["state"])[s["slots"].long()] if case["states"] else x.new_zeros(n, case["channels"])
    h, before, left, a = _steps(x, f, bias, comp, lengths, state)
    if case["op"] == "prompt":
        if case["states"]:
            whole = d(s["state"])
            whole[s["slots"].long()] = left
            left = whole
        return dict(h=h, state=left)
    if case["keep"]:  # from the state before every SEGMENT-th token of a sequence
        x, f = _kept(x), _kept(f)
        pieces = _segments(lengths)
        starts = torch.tensor([0] + pieces, device=DEVICE).cumsum(0)[:-1]
        _, before, _, a = _steps(x, f, bias, comp, pieces, before[starts])
    dh = d(s["dh"])
    G = d(s["dstate"]) if case["states"] else torch.zeros_like(state)  # of the state after the token at hand
    dx, df = torch.zeros_like(x), torch.zeros_like(x)
    for at, row in reversed(list(_walk(lengths))):
        now = G[at] + dh[row]
        dx[row] = (1 - a[row]) * now if comp else now
        df[row] = now * a[row] * (1 - a[row]) * (before[row] - x[row] if comp else before[row])
        G[at] = a[row] * now
    out = dict(h=h, dx=dx, df=df, dbias=df.sum(0))
    return dict(out, dstate=G) if case["states"] else out
