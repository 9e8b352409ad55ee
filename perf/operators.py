"""Cases of the sequence operators: the query/key norm with its rotation, and decayed linear attention.

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
CHUNK = 128  # tokens a chunk of the plain chunked form


def listed():
    return [
        # one new token of 24 running requests: the call's own latency counts
        dict(name="qk 24 tokens", op="qk", tokens=24, q_heads=16, k_heads=4, dim=128, rotary=128,
             axes=1, interleaved=False, dtype="bf16"),
        # patches of a short video: three position axes, part of the head rotated, odd count
        dict(name="qk video", op="qk", tokens=6137, q_heads=12, k_heads=12, dim=96, rotary=72,
             axes=3, interleaved=True, dtype="f32"),
        # a long prompt of a model with grouped heads
        dict(name="qk prompt", op="qk", tokens=16384, q_heads=32, k_heads=8, dim=128, rotary=128,
             axes=1, interleaved=False, dtype="bf16"),
        # the backward pass of a training batch
        dict(name="qk gradients", op="qk_grad", tokens=8192, q_heads=32, k_heads=8, dim=128, rotary=128,
             axes=1, interleaved=False, dtype="bf16"),
        # decoding a handful of requests
        dict(name="step 3 requests", op="step", requests=3, q_heads=16, kv_heads=16, key_dim=64,
             value_dim=64, dtype="bf16"),
        # decoding a full batch: the states are the traffic
        dict(name="step 192 requests", op="step", requests=192, q_heads=32, kv_heads=32, key_dim=128,
             value_dim=128, dtype="bf16"),
        # one short prompt
        dict(name="prompt short", op="prompt", tokens=333, seqs=1, q_heads=16, kv_heads=16, key_dim=128,
             value_dim=128, states=False, dtype="bf16"),
        # prompts of many requests packed together, continued from and written to their state slots
        dict(name="prompts packed", op="prompt", tokens=9001, seqs=11, q_heads=32, kv_heads=8, key_dim=128,
             value_dim=128, states=True, dtype="bf16"),
        # one long document: few heads, so the time axis has to be split
        dict(name="prompt long", op="prompt", tokens=49152, seqs=1, q_heads=16, kv_heads=16, key_dim=128,
             value_dim=128, states=False, dtype="bf16"),
        # the same operator in the framework's own type
        dict(name="prompts f32", op="prompt", tokens=2500, seqs=3, q_heads=12, kv_heads=12, key_dim=64,
             value_dim=64, states=True, dtype="f32"),
        # gradients of a training batch of equal sequences
        dict(name="gradients", op="grad", tokens=8192, seqs=4, q_heads=16, kv_heads=16, key_dim=128,
             value_dim=128, states=False, dtype="bf16"),
        # gradients of ragged sequences, grouped heads, uneven widths, with those of the states
        dict(name="gradients ragged", op="grad", tokens=1501, seqs=5, q_heads=8, kv_heads=2, key_dim=80,
             value_dim=48, states=True, dtype="f32"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["qk", "qk_grad", "step", "prompt", "prompt", "grad"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 1, 2, 4])
    if op in ("qk", "qk_grad"):
        dim = rng.choice([32, 64, 80, 96, 128, 192, 256])
        axes = rng.choice([1, 1, 2, 3])
        rotary = rng.choice([dim, dim, dim // 2])
        most = 8192 * 40 * 128 // (kv * (group + 1) * dim)
        return dict(op=op, tokens=_log_uniform(rng, 1, min(most, 40000)), q_heads=kv * group, k_heads=kv,
                    dim=dim, rotary=rotary, axes=axes, interleaved=rng.random() < 0.5, dtype=dtype)
    widths = [32, 40, 64, 80, 96, 128, 128]
    dk, dv = rng.choice(widths), rng.choice(widths)
    base = dict(op=op, q_heads=kv * group, kv_heads=kv, key_dim=dk, value_dim=dv, dtype=dtype)
    if op == "step":
        most = 192 * 32 * 128 * 128 // (kv * group * dk * dv)
        return dict(base, requests=_log_uniform(rng, 1, min(most, 512)))
    most = (16 * 49152 if op == "prompt" and dtype == "bf16" else 16 * 8192) // (kv * group)
    tokens = _log_uniform(rng, 1, min(most, 49152))
    return dict(base, tokens=tokens, seqs=min(tokens, _log_uniform(rng, 1, 32)), states=rng.random() < 0.5)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _lengths(case):
    """Ragged lengths with the case's total; equal ones for a training batch without states."""
    n, total = case["seqs"], case["tokens"]
    if case["op"] == "grad" and not case["states"] and total % n == 0:
        return [total // n] * n
    cut = random.Random(total * 131 + n)
    cuts = sorted(cut.randint(0, total) for _ in range(n - 1))
    if n >= 4:
        cuts[1] = cuts[0]  # an empty sequence among them
    if n >= 5:
        cuts[3] = max(cuts[2], min(cuts[2] + 1, total))  # and one of a single token
        cuts.sort()
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _sections(case):
    pairs, axes = case["rotary"] // 2, case["axes"]
    first = [pairs // axes] * axes
    first[0] += pairs - sum(first)
    return first


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _dtype(case)

    def normal(*shape, t=None):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(t or dtype)

    s = dict(case=case)
    if case["op"] in ("qk", "qk_grad"):
        T, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
        rows = normal(T, (hq + 2 * hk) * d)  # a projection's packed rows: queries, keys, values
        s["q"] = rows[:, :hq * d].view(T, hq, d)
        s["k"] = rows[:, hq * d:(hq + hk) * d].view(T, hk, d)
        s["wq"] = 1 + 0.2 * normal(d, t=torch.float32)
        s["wk"] = 1 + 0.2 * normal(d, t=torch.float32)
        if case["axes"] == 1:  # consecutive tokens at some depth of a long text
            first = torch.randint(0, 100000, (1,), generator=gen, device=DEVICE)
            s["positions"] = (first + torch.arange(T, device=DEVICE)).to(torch.int32).view(1, T)
        else:  # coordinates on a grid
            s["positions"] = torch.randint(0, 500, (case["axes"], T), generator=gen, device=DEVICE, dtype=torch.int32)
        if case["op"] == "qk_grad":
            s["gq"], s["gk"] = normal(T, hq, d), normal(T, hk, d)
        return s
    hq, hk, dk, dv = case["q_heads"], case["kv_heads"], case["key_dim"], case["value_dim"]
    # decay rates spread over the heads from fast to slow, as such models fix them
    rate = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEVICE, dtype=torch.float32) / hq)
    s["log_decay"] = -rate * (0.9 + 0.1 * torch.rand(hq, generator=gen, device=DEVICE))
    T = case["requests"] if case["op"] == "step" else case["tokens"]
    rows = normal(T, (hk * dv + hk * dk))  # keys come from the norm's pass, values lie in packed rows
    s["q"], s["k"] = normal(T, hq, dk), normal(T, hk, dk)
    s["v"] = rows[:, hk * dk:].view(T, hk, dv)
    if case["op"] == "step":
        slots = T + 3
        s["state"] = normal(slots, hq, dk, dv, t=torch.float32)
        s["slots"] = torch.randperm(slots, generator=gen, device=DEVICE)[:T].to(torch.int32)
        return s
    n = case["seqs"]
    s["lengths"] = _lengths(case)
    ends = torch.tensor([0] + s["lengths"]).cumsum(0)
    s["cu_seqlens"] = ends.to(torch.int32).to(DEVICE)
    if case["states"]:
        s["state"] = normal(n + 2, hq, dk, dv, t=torch.float32)
        s["slots"] = torch.randperm(n + 2, generator=gen, device=DEVICE)[:n].to(torch.int32)
    if case["op"] == "grad":
        s["do"] = normal(T, hq, dv)
        if case["states"]:
            s["state"] = s["state"][:n].contiguous()
            s["dstate"] = normal(n, hq, dk, dv, t=torch.float32)
    return s


# ---- the framework's operators ---------------------------------------------------


@functools.lru_cache(maxsize=None)
def _operator(op, dtype, *sizes):
    from tensoroperations_b200 import sequence
    if op == "qk":
        q_heads, k_heads, dim, rotary, interleaved, *sections = sizes
        return sequence.QkNormRotary(dtype, q_heads, k_heads, dim, rotary, sections, interleaved)
    return sequence.LinearAttention(dtype, *sizes)


def _run_own(s):
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] in ("qk", "qk_grad"):
        op = _operator("qk", case["dtype"], case["q_heads"], case["k_heads"], case["dim"], case["rotary"],
                       case["interleaved"], *_sections(case))
        q, k = torch.empty_like(s["q"], memory_format=torch.contiguous_format), \
            torch.empty_like(s["k"], memory_format=torch.contiguous_format)
        if case["op"] == "qk":
            op.forward(s["q"], s["k"], s["positions"], s["wq"], s["wk"], q, k, stream=stream)
            return dict(q=q, k=k)
        wq, wk = torch.empty_like(s["wq"]), torch.empty_like(s["wk"])
        ws = torch.empty(op.workspace_bytes(case["tokens"]), dtype=torch.uint8, device=DEVICE)
        op.backward(s["q"], s["k"], s["positions"], s["wq"], s["wk"], s["gq"], s["gk"], q, k, wq, wk, ws,
                    stream=stream)
        return dict(dq=q, dk=k, dwq=wq, dwk=wk)
    op = _operator("attention", case["dtype"], case["q_heads"], case["kv_heads"], case["key_dim"],
                   case["value_dim"])
    q, k, v, g = s["q"], s["k"], s["v"], s["log_decay"]
    T = q.shape[0]
    if case["op"] == "step":
        o = torch.empty(T, case["q_heads"], case["value_dim"], dtype=q.dtype, device=DEVICE)
        op.step(q, k, v, g, s["state"], o, slots=s["slots"], stream=stream)
        return dict(o=o, state=s["state"])
    if case["op"] == "prompt":
        o = torch.empty(T, case["q_heads"], case["value_dim"], dtype=q.dtype, device=DEVICE)
        ws = torch.empty(op.workspace_bytes(T, case["seqs"]), dtype=torch.uint8, device=DEVICE)
        if case["states"]:
            op.forward(q, k, v, g, s["cu_seqlens"], o, state_in=s["state"], state_out=s["state"],
                       slots=s["slots"], workspace=ws, stream=stream)
            return dict(o=o, state=s["state"])
        state = torch.empty(case["seqs"], case["q_heads"], case["key_dim"], case["value_dim"], device=DEVICE)
        op.forward(q, k, v, g, s["cu_seqlens"], o, state_out=state, workspace=ws, stream=stream)
        return dict(o=o, state=state)
    dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    ws = torch.empty(op.backward_workspace_bytes(T, case["seqs"]), dtype=torch.uint8, device=DEVICE)
    if case["states"]:
        dstate = torch.empty_like(s["state"])
        op.backward(q, k, v, g, s["cu_seqlens"], s["do"], dq, dk, dv, state_in=s["state"],
                    dstate_out=s["dstate"], dstate_in=dstate, workspace=ws, stream=stream)
        return dict(dq=dq, dk=dk, dv=dv, dstate=dstate)
    op.backward(q, k, v, g, s["cu_seqlens"], s["do"], dq, dk, dv, workspace=ws, stream=stream)
    return dict(dq=dq, dk=dk, dv=dv)


# ---- plain forms -----------------------------------------------------------------


def _angles(s, dtype):
    """cos and sin [T, 1, pairs]; the products of large positions need 64 bits to keep their fraction."""
    case = s["case"]
    pairs = case["rotary"] // 2
    freq = 10000.0 ** (-2.0 * torch.arange(pairs, device=DEVICE, dtype=torch.float64) / case["rotary"])
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=DEVICE),
                                   torch.tensor(_sections(case), device=DEVICE), output_size=pairs)
    angle = s["positions"][axis].t().to(torch.float64) * freq
    return angle.cos().to(dtype)[:, None], angle.sin().to(dtype)[:, None]


def _turn(x, cos, sin, rotary, interleaved):
    part, rest = x[..., :rotary], x[..., rotary:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.split(rotary // 2, -1)
    c, d = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((part, rest), -1)


def _norm_rotate(x, w, cos, sin, case):
    n = x * ((x * x).mean(-1, keepdim=True) + 1e-6).rsqrt()
    return _turn(n * w, cos, sin, case["rotary"], case["interleaved"])


def _norm_rotate_grad(x, w, g, cos, sin, case):
    r = ((x * x).mean(-1, keepdim=True) + 1e-6).rsqrt()
    n, u = x * r, _turn(g, cos, -sin, case["rotary"], case["interleaved"])
    d = u * w
    return r * (d - n * (d * n).mean(-1, keepdim=True)), (u * n).sum((0, 1))


def _chunks(lengths):
    """Row numbers [chunks, CHUNK] of the packed tokens (-1: none), each chunk's sequence and first token in it."""
    n = torch.tensor(lengths, device=DEVICE)
    count = (n + CHUNK - 1) // CHUNK
    total = sum(-(-x // CHUNK) for x in lengths)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=DEVICE), count, output_size=total)
    first = (torch.arange(total, device=DEVICE) - (count.cumsum(0) - count)[seq]) * CHUNK
    at = first[:, None] + torch.arange(CHUNK, device=DEVICE)
    row = torch.where(at < n[seq][:, None], at + (n.cumsum(0) - n)[seq][:, None], -1)
    return row, seq, first


def _chain(a, b, c, g, lengths, state, backwards=False):
    """sum_j l^(i-j) (a_i.b_j) c_j over the earlier tokens j <= i of each sequence (later ones if
    `backwards`), with `state` [seqs, heads, b, c] entering (forwards it decays once more before the first
    token); and the state left at the other end.  a, b, c: [tokens, heads, width]."""
    if backwards:  # the same with each packed sequence read from its end
        m, state = _chain(a.flip(0), b.flip(0), c.flip(0), g, lengths[::-1],
                          (state * (-g).exp()[:, None, None]).flip(0))
        return m.flip(0), (state * g.exp()[:, None, None]).flip(0)
    row, seq, first = _chunks(lengths)
    there = (row >= 0)[:, None, :, None]
    x, y, z = (t[row.clamp(min=0)].transpose(1, 2) * there for t in (a, b, c))  # [chunks, heads, CHUNK, width]
    i = torch.arange(CHUNK, device=DEVICE, dtype=g.dtype)
    count = (row >= 0).sum(1).to(g.dtype)  # tokens of each chunk
    gap = i[:, None] - i
    mask = torch.where(gap >= 0, (g[:, None, None] * gap.clamp(min=0)).exp(), 0.0)
    out = (x @ y.transpose(-1, -2) * mask) @ z
    left = (g[None, :, None] * (count[:, None, None] - 1 - i).clamp(min=0)).exp()
    adds = (y * left[..., None]).transpose(-1, -2) @ z  # [chunks, heads, b, c]
    # what each chunk's additions, and the entering state, amount to before every chunk
    start, end = first.to(g.dtype), first.to(g.dtype) + count
    before = (seq[:, None] == seq) & (first[:, None] > first)
    apart = (start[:, None] - end).clamp(min=0)
    weigh = torch.where(before, (g[:, None, None] * apart).exp(), 0.0)  # [heads, chunks, chunks]
    n, h = adds.shape[:2]
    entering = (weigh @ adds.transpose(0, 1).reshape(h, n, -1)).view(h, n, *adds.shape[2:]).transpose(0, 1)
    entering = entering + state[seq] * (g[None, :] * start[:, None]).exp()[..., None, None]
    out = out + (x @ entering) * (g[:, None] * (i + 1)).exp()[None, :, :, None]
    size = torch.tensor(lengths, device=DEVICE, dtype=g.dtype)
    weigh = torch.where(seq == torch.arange(len(lengths), device=DEVICE)[:, None],
                        (g[:, None, None] * (size[:, None] - end).clamp(min=0)).exp(), 0.0)
    leaving = (weigh @ adds.transpose(0, 1).reshape(h, n, -1)).view(h, -1, *adds.shape[2:]).transpose(0, 1)
    leaving = leaving + state * (g[None, :] * size[:, None]).exp()[..., None, None]
    return out.transpose(1, 2)[row >= 0], leaving


def _run_plain(s):
    case = s["case"]
    f = lambda x: x.to(torch.float32)  # noqa: E731
    if case["op"] in ("qk", "qk_grad"):
        cos, sin = _angles(s, torch.float32)
        if case["op"] == "qk":
            return {n: _norm_rotate(f(s[n]), s["w" + n], cos, sin, case).to(s[n].dtype) for n in ("q", "k")}
        dq, dwq = _norm_rotate_grad(f(s["q"]), s["wq"], f(s["gq"]), cos, sin, case)
        dk, dwk = _norm_rotate_grad(f(s["k"]), s["wk"], f(s["gk"]), cos, sin, case)
        return dict(dq=dq.to(s["q"].dtype), dk=dk.to(s["k"].dtype), dwq=dwq, dwk=dwk)
    g, dtype = s["log_decay"], s["q"].dtype
    group = case["q_heads"] // case["kv_heads"]
    scale = case["key_dim"] ** -0.5
    q = f(s["q"])
    k, v = (f(s[n]).repeat_interleave(group, 1) for n in ("k", "v"))
    if case["op"] == "step":
        at = s["slots"].long()
        state = s["state"][at] * g.exp()[:, None, None] + k[..., None] * v[..., None, :]
        s["state"][at] = state
        return dict(o=(scale * (q[..., None] * state).sum(-2)).to(dtype), state=s["state"])
    n = case["seqs"]
    none = torch.zeros(n, case["q_heads"], case["key_dim"], case["value_dim"], device=DEVICE)
    if case["op"] == "prompt":
        at = s["slots"].long() if case["states"] else None
        o, state = _chain(q, k, v, g, s["lengths"], none if at is None else s["state"][at])
        if at is not None:
            s["state"][at] = state
            state = s["state"]
        return dict(o=(scale * o).to(dtype), state=state)
    do = f(s["do"])
    state, dstate = (s["state"], s["dstate"]) if case["states"] else (none, none)
    dq, _ = _chain(do, v, k, g, s["lengths"], state.transpose(-1, -2))
    dv, left = _chain(k, q * scale, do, g, s["lengths"], dstate, backwards=True)
    dk, _ = _chain(v, do, q * scale, g, s["lengths"], dstate.transpose(-1, -2), backwards=True)
    dk, dv = (x.view(x.shape[0], -1, group, x.shape[-1]).sum(2) for x in (dk, dv))
    out = dict(dq=(scale * dq).to(dtype), dk=dk.to(dtype), dv=dv.to(dtype))
    return dict(out, dstate=left) if case["states"] else out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("qk", "qk_grad"):
        T, d, heads = case["tokens"], case["dim"], case["q_heads"] + case["k_heads"]
        passes = 2 if case["op"] == "qk" else 3
        more = 4 * T * case["axes"] + 8 * d * (1 if case["op"] == "qk" else 2)
        return dict(bytes=passes * T * heads * d * size + more,
                    flops=(8 if case["op"] == "qk" else 16) * T * heads * d)
    hq, hk, dk, dv = case["q_heads"], case["kv_heads"], case["key_dim"], case["value_dim"]
    one = 4 * hq * dk * dv  # bytes of one sequence's states
    T = case["requests"] if case["op"] == "step" else case["tokens"]
    rows = T * (hq * (dk + dv) + hk * (dk + dv)) * size
    if case["op"] == "step":
        return dict(bytes=rows + 2 * T * one, flops=4 * T * hq * dk * dv)
    states = case["seqs"] * one * (2 if case["states"] else 1)
    if case["op"] == "prompt":
        return dict(bytes=rows + states, flops=4 * T * hq * dk * dv)
    rows += T * (hq * dk + hk * (dk + dv)) * size
    return dict(bytes=rows + (3 * case["seqs"] * one if case["states"] else 0), flops=10 * T * hq * dk * dv)


# ---- the definitions, token by token, in 64 bits -------------------------------------


def _walk(lengths):
    """For each time step, the sequences that have such a token, and its packed row."""
    first = [sum(lengths[:n]) for n in range(len(lengths))]
    length, first = torch.tensor(lengths, device=DEVICE), torch.tensor(first, device=DEVICE)
    order = torch.argsort(length, descending=True)
    ordered = sorted(lengths, reverse=True)
    live = len(lengths)
    for t in range(max(lengths, default=0)):
        while live and ordered[live - 1] <= t:
            live -= 1
        yield order[:live], first[order[:live]] + t, live


def _scan(q, k, v, lam, lengths, state):
    """S <- l S + k v^T; o = S^T q at every token.  `state` is left as it is."""
    order = torch.argsort(torch.tensor(lengths, device=DEVICE), descending=True)
    S = state[order].clone()  # longest first, so that the live ones lead
    o = q.new_zeros(q.shape[0], q.shape[1], v.shape[-1])
    for _, row, live in _walk(lengths):
        part = S[:live]
        part *= lam[:, None, None]
        part += k[row][..., None] * v[row][..., None, :]
        o[row] = (q[row][..., None, :] @ part)[..., 0, :]
    left = torch.empty_like(S)
    left[order] = S
    return o, left


def exact(case, seed):
    s = prepare(case, seed)
    w = lambda n: s[n].to(torch.float64)  # noqa: E731
    if case["op"] in ("qk", "qk_grad"):
        pairs = case["rotary"] // 2
        owner = [a for a, n in enumerate(_sections(case)) for _ in range(n)]
        first = [2 * j if case["interleaved"] else j for j in range(pairs)]
        second = [2 * j + 1 if case["interleaved"] else j + pairs for j in range(pairs)]
        angle = torch.stack([w("positions")[owner[j]] * math.exp(-2.0 * j / case["rotary"] * math.log(10000.0))
                             for j in range(pairs)], 1)[:, None]
        out = {}
        for n in ("q", "k"):
            x, weight = w(n), w("w" + n)
            length = (x.square().sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt()
            if case["op"] == "qk":
                y = x / length * weight
                z = y.clone()
                z[..., first] = y[..., first] * angle.cos() - y[..., second] * angle.sin()
                z[..., second] = y[..., first] * angle.sin() + y[..., second] * angle.cos()
                out[n] = z
                continue
            z = w("g" + n)
            u = z.clone()
            u[..., first] = z[..., first] * angle.cos() + z[..., second] * angle.sin()
            u[..., second] = z[..., second] * angle.cos() - z[..., first] * angle.sin()
            out["dw" + n] = (u * x / length).sum(0).sum(0)
            d = u * weight
            out["d" + n] = d / length - x * (d * x).sum(-1, keepdim=True) / (case["dim"] * length ** 3)
        return out
    lam = w("log_decay").exp()
    group = case["q_heads"] // case["kv_heads"]
    heads = torch.arange(case["q_heads"], device=DEVICE) // group
    scale = 1.0 / math.sqrt(case["key_dim"])
    q, k, v = w("q"), w("k")[:, heads], w("v")[:, heads]
    if case["op"] == "step":
        state = w("state")
        for r, slot in enumerate(s["slots"].tolist()):
            state[slot] = lam[:, None, None] * state[slot] + k[r][..., None] * v[r][..., None, :]
        o = torch.einsum("rhk,rhkv->rhv", q, state[s["slots"].long()])
        return dict(o=scale * o, state=state)
    n, lengths = case["seqs"], s["lengths"]
    zero = torch.zeros(n, case["q_heads"], case["key_dim"], case["value_dim"], device=DEVICE, dtype=torch.float64)
    if case["op"] == "prompt":
        o, state = _scan(q, k, v, lam, lengths, w("state")[s["slots"].long()] if case["states"] else zero)
        if case["states"]:
            whole = w("state")
            whole[s["slots"].long()] = state
            state = whole
        return dict(o=scale * o, state=state)
    state, dstate = (w("state"), w("dstate")) if case["states"] else (zero, zero.clone())
    do = w("do")
    dq, _ = _scan(do, v, k, lam, lengths, state.transpose(-1, -2))
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    order = torch.argsort(torch.tensor(lengths, device=DEVICE), descending=True)
    G = dstate[order].clone()  # the gradient with respect to the state after the token at hand
    for _, row, live in reversed(list(_walk(lengths))):
        part = G[:live]
        part += scale * q[row][..., None] * do[row][..., None, :]
        dk[row] = (part @ v[row][..., None])[..., 0]
        dv[row] = (k[row][..., None, :] @ part)[..., 0, :]
        part *= lam[:, None, None]
    left = torch.empty_like(G)
    left[order] = G
    shared = lambda x: x.view(x.shape[0], -1, group, x.shape[-1]).sum(2)  # noqa: E731
    out = dict(dq=scale * dq, dk=shared(dk), dv=shared(dv))
    return dict(out, dstate=left) if case["states"] else out
