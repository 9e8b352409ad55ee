"""The sequence operators on the GPU against token-by-token definitions in float64.

Tolerances (relative 2-norm), from the types alone:
* f32 results: 2e-6.  A rounding is at most 2^-24 = 6e-8; every value is a sum of
  a few hundred products whose roundings add in quadrature (16 x 6e-8 = 1e-6) plus
  a decay factor from expf (2 ulp) whose argument is rounded once.
* bf16 results: 2^-8.  A rounding to 8 bits is half a spacing at most, 2^-9.2 of the
  values in the mean square; products of bf16 rows go through one more bf16 operand,
  so there are two, in quadrature 2^-8.7.
* one value: 16 times that, relative to the larger of itself and the rms (a value's
  own error is not averaged).
"""
import math

import pytest

from tensoroperations_b200 import abi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOL = {"f32": 2e-6, "bf16": 2.0 ** -8}
KIND = {"f32": torch.float32, "bf16": torch.bfloat16}


def close(got, ref, tol, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    got, ref = got.double(), ref.double()
    if not ref.numel():
        return
    assert torch.isfinite(got).all(), what
    d, norm = got - ref, ref.norm()
    assert d.norm() <= tol * norm, (what, float(d.norm() / norm), tol)
    rms = norm / math.sqrt(ref.numel())
    worst = (d.abs() / torch.maximum(ref.abs(), rms).clamp(min=1e-300)).max()
    assert worst <= 16 * tol, (what, float(worst))


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(gen, shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda").to(KIND[dtype])


# ---- query / key norm with rotation ------------------------------------------------


def qk_definition(x, w, pos, rotary, sections, interleaved, theta=10000.0, eps=1e-6):
    """y, and the function of x in float64."""
    x = x.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = n * (1.0 if w is None else w.double())
    out = y.clone()
    axis = 0
    left = list(sections)
    for j in range(rotary // 2):
        while left[axis] == 0:
            axis += 1
        left[axis] -= 1
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rotary // 2)
        ang = pos[axis].double() * theta ** (-2.0 * j / rotary)
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
    return out


QK = [
    # dtype, tokens, q heads, k heads, head_dim, rotary, sections, interleaved
    ("bf16", 1, 16, 4, 128, 128, [64], False),
    ("bf16", 37, 5, 3, 128, 128, [64], False),
    ("bf16", 700, 8, 2, 128, 128, [64], True),
    ("f32", 33, 3, 1, 128, 128, [64], False),
    ("f32", 129, 4, 4, 96, 72, [12, 12, 12], True),
    ("bf16", 65, 6, 2, 96, 48, [8, 10, 6], False),
    ("bf16", 19, 2, 1, 80, 40, [5, 5, 5, 5], False),
    ("f32", 50, 2, 2, 256, 256, [128], True),
    ("bf16", 50, 2, 2, 256, 256, [128], False),
    ("bf16", 17, 3, 1, 192, 64, [32], True),
    ("f32", 9, 1, 1, 2, 2, [1], False),
    ("bf16", 9, 3, 1, 6, 6, [3], True),
    ("bf16", 21, 2, 1, 130, 66, [33], False),
    ("f32", 21, 2, 1, 202, 0, [0], False),
    ("bf16", 5, 40, 40, 64, 64, [64 // 2], False),
]


def qk_inputs(dtype, T, hq, hk, D, axes, seed=1, spread=5000):
    g = rng(seed)
    rows = normal(g, (T, (hq + 2 * hk) * D), dtype)
    q, k = rows[:, :hq * D].view(T, hq, D), rows[:, hq * D:(hq + hk) * D].view(T, hk, D)
    pos = torch.randint(0, spread, (axes, T), generator=g, device="cuda", dtype=torch.int32)
    wq, wk = (1 + 0.2 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    return q, k, pos, wq, wk


@pytest.mark.parametrize("dtype,T,hq,hk,D,rot,sections,inter", QK)
def test_qk_forward(dtype, T, hq, hk, D, rot, sections, inter):
    from tensoroperations_b200 import sequence
    q, k, pos, wq, wk = qk_inputs(dtype, T, hq, hk, D, len(sections))
    op = sequence.QkNormRotary(dtype, hq, hk, D, rot, sections, inter)
    yq, yk = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
    op.forward(q, k, pos, wq, wk, yq, yk)
    close(yq, qk_definition(q, wq, pos, rot, sections, inter), TOL[dtype], "q")
    close(yk, qk_definition(k, wk, pos, rot, sections, inter), TOL[dtype], "k")
    # in place, and without weights
    ref = qk_definition(q, None, pos, rot, sections, inter)
    keep = k.clone()
    op.forward(q, k, pos, None, None, q, yk)
    close(q, ref, TOL[dtype], "q in place")
    assert torch.equal(k, keep)
    close(yk, qk_definition(k, None, pos, rot, sections, inter), TOL[dtype], "k without weights")


@pytest.mark.parametrize("dtype,T,hq,hk,D,rot,sections,inter", QK)
def test_qk_backward(dtype, T, hq, hk, D, rot, sections, inter):
    from tensoroperations_b200 import sequence
    q, k, pos, wq, wk = qk_inputs(dtype, T, hq, hk, D, len(sections), seed=2)
    g = rng(3)
    gq, gk = normal(g, (T, hq, D), dtype), normal(g, (T, hk, D), dtype)
    op = sequence.QkNormRotary(dtype, hq, hk, D, rot, sections, inter)
    dq, dk = torch.empty_like(gq), torch.empty_like(gk)
    dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
    ws = torch.empty(op.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    op.backward(q, k, pos, wq, wk, gq, gk, dq, dk, dwq, dwk, ws)
    for x, w, gy, dx, dw, name in ((q, wq, gq, dq, dwq, "q"), (k, wk, gk, dk, dwk, "k")):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y = qk_definition(x64, w64, pos, rot, sections, inter)
        rx, rw = torch.autograd.grad((y * gy.double()).sum(), (x64, w64))
        close(dx, rx, TOL[dtype], "d" + name)
        close(dw, rw, TOL["f32"] * 2, "dw" + name)  # sums over all rows: longer than a row's
        # against differences of the definition, along one direction
        v = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-6
        f = [(qk_definition(x.double() + sgn * h * v, w, pos, rot, sections, inter) * gy.double()).sum()
             for sgn in (1, -1)]
        slope = float((f[0] - f[1]) / (2 * h))
        size = float(dx.double().norm() * v.norm())
        assert abs(float((dx.double() * v).sum()) - slope) <= (TOL[dtype] + 1e-6) * size
    # gradients in place of the incoming ones, and no weight gradients
    op.backward(q, k, pos, wq, wk, gq, gk, gq, gk, None, None, ws)
    assert torch.equal(gq, dq) and torch.equal(gk, dk)


def test_qk_positions_keep_their_fraction():
    """Positions up to the int32 limits, negative ones too, at f32 accuracy."""
    from tensoroperations_b200 import sequence
    pos = torch.tensor([[2**31 - 1, -2**31, 10**9 + 7, -123456789, 0, 1, 99999]], dtype=torch.int32, device="cuda")
    T, D = pos.shape[1], 64
    q = normal(rng(5), (T, 2, D), "f32")
    op = sequence.QkNormRotary("f32", 2, 2, D)
    yq, yk = torch.empty_like(q), torch.empty_like(q)
    op.forward(q, q, pos, None, None, yq, yk)
    # the definition's own angles in float64 are good to 2^31 * 2^-53 = 2.4e-7 radians
    close(yq, qk_definition(q, None, pos, D, [D // 2], False), TOL["f32"])
    assert torch.equal(yq, yk)


def test_qk_odd_addresses_zero_rows_and_no_tokens():
    from tensoroperations_b200 import sequence
    T, D = 23, 64
    raw = normal(rng(6), (T * 3 * D + 1,), "bf16")
    q = raw[1:].view(T, 3, D)  # two bytes off: single values
    pos = torch.arange(T, dtype=torch.int32, device="cuda").view(1, T)
    op = sequence.QkNormRotary("bf16", 3, 1, D)
    yq, yk = torch.empty(T, 3, D, dtype=torch.bfloat16, device="cuda"), torch.empty(T, 1, D, dtype=torch.bfloat16, device="cuda")
    q[3] = 0
    op.forward(q, q[:, :1], pos, None, None, yq, yk)
    close(yq, qk_definition(q, None, pos, D, [32], False), TOL["bf16"])
    assert (yq[3] == 0).all() and torch.equal(yk, yq[:, :1])
    inter = sequence.QkNormRotary("bf16", 3, 1, D, interleaved=True)
    with pytest.raises(abi.ToError) as e:
        inter.forward(q, q[:, :1], pos, None, None, yq, yk)
    assert e.value.status == abi.TO_ERR_ALIGNMENT
    op.forward(q[:0], q[:0, :1], pos[:, :0].contiguous(), None, None, yq[:0], yk[:0])
    w = torch.full((D,), float("nan"), device="cuda")
    ws = torch.empty(op.workspace_bytes(0), dtype=torch.uint8, device="cuda")
    op.backward(q[:0], q[:0, :1], pos[:, :0].contiguous(), None, None, yq[:0], yk[:0], yq[:0], yk[:0], w, None, ws)
    assert (w == 0).all()


# ---- linear attention ----------------------------------------------------------------


def attention_definition(q, k, v, decay, lengths, scale, state):
    """o and the states left, token by token, in float64."""
    group = q.shape[1] // k.shape[1]
    k, v = k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    q, lam = q.double(), decay.double().clamp(max=0).exp()[:, None, None]
    o, left, t = [], [], 0
    for n, length in enumerate(lengths):
        S = state[n].double()
        for _ in range(length):
            S = lam * S + k[t][..., None] * v[t][..., None, :]
            o.append(scale * (q[t][..., None, :] @ S)[..., 0, :])
            t += 1
        left.append(S)
    o = torch.stack(o) if o else q.new_zeros(0, q.shape[1], v.shape[-1])
    return o, torch.stack(left)


def attention_inputs(dtype, lengths, hq, hk, dk, dv, seed=1):
    g = rng(seed)
    T = sum(lengths)
    q = normal(g, (T, hq, dk), dtype)
    rows = normal(g, (T, hk * (dk + dv)), dtype)  # keys and values packed in one row
    k, v = rows[:, :hk * dk].view(T, hk, dk), rows[:, hk * dk:].view(T, hk, dv)
    decay = -2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)
    cu = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
    return q, k, v, decay, cu


def scratch(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda").fill_(0xff) if n else None


LA = [
    # dtype, lengths, q heads, kv heads, key dim, value dim
    ("f32", [1], 1, 1, 1, 1),
    ("f32", [5, 0, 1, 64, 65, 127], 4, 2, 16, 24),
    ("f32", [130, 63], 3, 3, 64, 64),
    ("f32", [200], 2, 1, 128, 128),
    ("f32", [77, 3], 2, 2, 256, 40),
    ("f32", [90], 2, 2, 40, 256),
    ("f32", [33], 2, 1, 13, 7),
    ("f32", [1500, 0, 700], 4, 1, 32, 48),  # several segments
    ("bf16", [1], 16, 4, 128, 128),
    ("bf16", [0, 127, 128, 0, 129, 1], 4, 2, 128, 128),
    ("bf16", [255, 257, 2], 6, 6, 64, 128),
    ("bf16", [300], 3, 1, 128, 64),
    ("bf16", [300, 11], 8, 8, 64, 64),
    ("bf16", [140, 5], 2, 2, 80, 96),
    ("bf16", [140, 5], 2, 1, 40, 32),
    ("bf16", [131], 2, 2, 13, 9),
    ("bf16", [150], 1, 1, 256, 200),
    ("bf16", [1537, 1, 0, 640], 4, 2, 128, 128),
    ("bf16", [2100], 2, 2, 64, 96),
]


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype,lengths,hq,hk,dk,dv", LA)
def test_attention_forward(dtype, lengths, hq, hk, dk, dv, states):
    from tensoroperations_b200 import sequence
    q, k, v, decay, cu = attention_inputs(dtype, lengths, hq, hk, dk, dv)
    n = len(lengths)
    op = sequence.LinearAttention(dtype, hq, hk, dk, dv)
    o = torch.full((q.shape[0], hq, dv), float("nan"), dtype=q.dtype, device="cuda")
    ws = scratch(op.workspace_bytes(q.shape[0], n))
    if states:
        pool = torch.randn(n + 3, hq, dk, dv, generator=rng(9), device="cuda")
        slots = torch.randperm(n + 3, generator=rng(10), device="cuda")[:n].to(torch.int32)
        before = pool.clone()
        op.forward(q, k, v, decay, cu, o, state_in=pool, state_out=pool, slots=slots, workspace=ws)
        ref, left = attention_definition(q, k, v, decay, lengths, dk ** -0.5, before[slots.long()])
        whole = before.double()
        whole[slots.long()] = left
        close(pool, whole, TOL["f32"], "states")
    else:
        left = torch.full((n, hq, dk, dv), float("nan"), device="cuda")
        op.forward(q, k, v, decay, cu, o, state_out=left, workspace=ws)
        ref, want = attention_definition(q, k, v, decay, lengths, dk ** -0.5, torch.zeros_like(left))
        close(left, want, TOL["f32"], "states")
    close(o, ref, TOL[dtype], "o")
    again = torch.empty_like(o)
    if not states:  # the same call gives the same bits, without the states too
        op.forward(q, k, v, decay, cu, again, state_out=left, workspace=ws)
        assert torch.equal(o, again)
        op.forward(q, k, v, decay, cu, again, workspace=ws)
        close(again, ref, TOL[dtype], "o without states")


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype,lengths,hq,hk,dk,dv", LA)
def test_attention_backward(dtype, lengths, hq, hk, dk, dv, states):
    from tensoroperations_b200 import sequence
    q, k, v, decay, cu = attention_inputs(dtype, lengths, hq, hk, dk, dv, seed=4)
    n, g = len(lengths), rng(5)
    do = normal(g, (q.shape[0], hq, dv), dtype)
    S = torch.randn(n, hq, dk, dv, generator=g, device="cuda")
    G = torch.randn(n, hq, dk, dv, generator=g, device="cuda")
    if not states:
        S, G = torch.zeros_like(S), torch.zeros_like(G)
    x = [t.double().requires_grad_() for t in (q, k, v, S)]
    o, left = attention_definition(x[0], x[1], x[2], decay, lengths, dk ** -0.5, x[3])
    ref = torch.autograd.grad((o * do.double()).sum() + (left * G.double()).sum(), x)
    op = sequence.LinearAttention(dtype, hq, hk, dk, dv)
    ws = scratch(op.backward_workspace_bytes(q.shape[0], n))
    dq, dk_, dv_ = (torch.full(t.shape, float("nan"), dtype=t.dtype, device="cuda") for t in (q, k, v))
    dS = torch.full_like(S, float("nan"))
    more = dict(state_in=S, dstate_out=G) if states else {}
    op.backward(q, k, v, decay, cu, do, dq, dk_, dv_, dstate_in=dS, workspace=ws, **more)
    for got, want, name in ((dq, ref[0], "dq"), (dk_, ref[1], "dk"), (dv_, ref[2], "dv")):
        close(got, want, TOL[dtype], name)
    close(dS, ref[3], TOL["f32"], "dstate")
    # against differences of the definition along one direction
    h, d = 1e-5, [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in x]
    with torch.no_grad():
        f = []
        for sgn in (1, -1):
            y = [t + sgn * h * e for t, e in zip(x, d)]
            o, left = attention_definition(y[0], y[1], y[2], decay, lengths, dk ** -0.5, y[3])
            f.append((o * do.double()).sum() + (left * G.double()).sum())
    slope = float((f[0] - f[1]) / (2 * h))
    got = sum(float((a.double() * e).sum()) for a, e in zip((dq, dk_, dv_, dS), d))
    size = sum(float(a.double().norm() * e.norm()) for a, e in zip((dq, dk_, dv_, dS), d))
    assert abs(got - slope) <= (TOL[dtype] + 1e-6) * size
    second = [torch.empty_like(t) for t in (dq, dk_, dv_)]
    op.backward(q, k, v, decay, cu, do, *second, workspace=ws, **more)
    close(second[0], ref[0], TOL[dtype], "dq without dstate")
    close(second[2], ref[2], TOL[dtype], "dv without dstate")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_decays(dtype):
    """No decay, a very slow, a strong and an instant one, and a positive value (counts as none)."""
    from tensoroperations_b200 import sequence
    lengths, dk = [300, 700], 64
    q, k, v, _, cu = attention_inputs(dtype, lengths, 6, 6, dk, dk, seed=7)
    decay = torch.tensor([0.0, -1e-7, -5.0, -300.0, -math.inf, 0.5], device="cuda")
    op = sequence.LinearAttention(dtype, 6, 6, dk, dk, scale=0.25)
    o = torch.empty_like(q)
    S = torch.randn(2, 6, dk, dk, generator=rng(8), device="cuda")
    left = torch.empty_like(S)
    ws = scratch(op.workspace_bytes(1000, 2))
    op.forward(q, k, v, decay, cu, o, state_in=S, state_out=left, workspace=ws)
    lam_safe = decay.clone()
    ref, want = attention_definition(q, k, v, lam_safe, lengths, 0.25, S)
    for h in range(6):  # head by head: their sizes differ
        close(o[:, h], ref[:, h], TOL[dtype], f"head {h}")
        close(left[:, h], want[:, h], TOL["f32"], f"state {h}")
    do = normal(rng(9), o.shape, dtype)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    dS = torch.empty_like(S)
    ws = scratch(op.backward_workspace_bytes(1000, 2))
    op.backward(q, k, v, decay, cu, do, *grads, state_in=S, dstate_out=left, dstate_in=dS, workspace=ws)
    x = [t.double().requires_grad_() for t in (q, k, v, S)]
    o2, l2 = attention_definition(x[0], x[1], x[2], lam_safe, lengths, 0.25, x[3])
    ref = torch.autograd.grad((o2 * do.double()).sum() + (l2 * left.double()).sum(), x)
    for h in range(6):
        for got, want in zip(grads, ref[:3]):
            close(got[:, h], want[:, h], TOL[dtype], f"gradient, head {h}")
        if h < 3:  # with stronger decays the entering state's gradient is nothing but tiny values
            close(dS[:, h], ref[3][:, h], 2 * TOL["f32"], f"dstate {h}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_nothing(dtype):
    """No tokens at all: empty sequences hand their states, and the states' gradients, on."""
    from tensoroperations_b200 import sequence
    op = sequence.LinearAttention(dtype, 4, 2, 64, 32)
    q, k, v, decay, cu = attention_inputs(dtype, [0, 0, 0], 4, 2, 64, 32)
    S, left = torch.randn(3, 4, 64, 32, generator=rng(1), device="cuda"), torch.empty(3, 4, 64, 32, device="cuda")
    o = torch.empty(0, 4, 32, dtype=q.dtype, device="cuda")
    op.forward(q, k, v, decay, cu, o, state_in=S, state_out=left, workspace=scratch(op.workspace_bytes(0, 3)))
    assert torch.equal(S, left)
    back = torch.empty_like(S)
    op.backward(q, k, v, decay, cu, o, q.clone(), k.clone(), v.clone(), state_in=S, dstate_out=left, dstate_in=back,
                workspace=scratch(op.backward_workspace_bytes(0, 3)))
    assert torch.equal(back, left)
    op.forward(q, k, v, decay, cu[:1].contiguous(), o)  # and no sequences
    op.step(q, k, v, decay, S, o)


def test_qk_without_keys():
    from tensoroperations_b200 import sequence
    q, _, pos, wq, _ = qk_inputs("bf16", 50, 3, 1, 64, 1)
    op = sequence.QkNormRotary("bf16", 3, 0, 64)
    none, y = q[:, :0], torch.empty(50, 3, 64, dtype=q.dtype, device="cuda")
    op.forward(q, none, pos, wq, None, y, none)
    close(y, qk_definition(q, wq, pos, 64, [32], False), TOL["bf16"])
    g, dq, dw = torch.randn_like(y), torch.empty_like(y), torch.empty_like(wq)
    ws = torch.empty(op.workspace_bytes(50), dtype=torch.uint8, device="cuda")
    op.backward(q, none, pos, wq, None, g, none, dq, none, dw, None, ws)
    x64 = q.double().requires_grad_()
    w64 = wq.double().requires_grad_()
    rx, rw = torch.autograd.grad((qk_definition(x64, w64, pos, 64, [32], False) * g.double()).sum(), (x64, w64))
    close(dq, rx, TOL["bf16"])
    close(dw, rw, 2 * TOL["f32"])


@pytest.mark.parametrize("tokens", [1, 3, 17, 32])
def test_attention_few_tokens_round_once(tokens):
    """From nothing, few tokens: the result's own rounding alone (half the spacing of bf16 values,
    2^-7 of the power of two below, and what two planes leave of P)."""
    from tensoroperations_b200 import sequence
    q, k, v, decay, cu = attention_inputs("bf16", [tokens], 4, 2, 128, 64, seed=31)
    op = sequence.LinearAttention("bf16", 4, 2, 128, 64)
    o = torch.empty(tokens, 4, 64, dtype=q.dtype, device="cuda")
    op.forward(q, k, v, decay, cu, o)
    ref, _ = attention_definition(q, k, v, decay, [tokens], 128 ** -0.5, torch.zeros(1, 4, 128, 64, device="cuda"))
    half = 0.5 * 2.0 ** (ref.abs().clamp(min=1e-30).log2().floor() - 7)
    assert ((o.double() - ref).abs() <= half + 2.0 ** -14 * ref.abs().amax(-1, True)).all()


def test_attention_long_prompts_repeat_to_the_bit():
    """Many chunks and segments, calls back to back on changing inputs: every call gives the same
    bits, and the right values (a warp that ran ahead of its group would show here)."""
    from tensoroperations_b200 import sequence
    T, H, d = 20000, 8, 128
    op = sequence.LinearAttention("bf16", H, H, d, d)
    sets = [attention_inputs("bf16", [T], H, H, d, d, seed=s) for s in (21, 22)]
    ws = scratch(op.workspace_bytes(T, 1))
    first = []
    for rep in range(40):
        q, k, v, decay, cu = sets[rep % 2]
        o, left = torch.empty_like(q), torch.empty(1, H, d, d, device="cuda")
        op.forward(q, k, v, decay, cu, o, state_out=left, workspace=ws)
        if rep < 2:
            first.append((o, left))
        elif rep % 7 == 0:
            assert torch.equal(o, first[rep % 2][0]) and torch.equal(left, first[rep % 2][1]), rep
    q, k, v, decay, cu = sets[0]
    ref, want = attention_definition(q, k, v, decay, [T], d ** -0.5, torch.zeros(1, H, d, d, device="cuda"))
    close(first[0][0], ref, TOL["bf16"])
    close(first[0][1], want, TOL["f32"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_other_rows_do_not_matter(dtype):
    """Rows between, before and after the sequences, and other sequences' rows, hold NaN and inf."""
    from tensoroperations_b200 import sequence
    dk, T = 128, 900
    q, k, v, decay, _ = attention_inputs(dtype, [T], 2, 2, dk, dk, seed=11)
    op = sequence.LinearAttention(dtype, 2, 2, dk, dk)
    # sequence 0: rows 40..239 poisoned; sequence 1: rows 240..539 clean; sequence 2: 540..649 poisoned
    q, k, v = q.clone(), k.clone(), v.clone()
    for t in (q, k, v):
        t[:240] = float("nan")
        t[540:] = float("inf")
    do = normal(rng(12), (T, 2, dk), dtype)
    do[:240] = float("nan")
    do[540:] = float("inf")
    cu = torch.tensor([40, 240, 540, 650], dtype=torch.int32, device="cuda")
    o = torch.full((T, 2, dk), 7.0, dtype=q.dtype, device="cuda")
    left = torch.empty(3, 2, dk, dk, device="cuda")
    op.forward(q, k, v, decay, cu, o, state_out=left, workspace=scratch(op.workspace_bytes(T, 3)))
    ref, want = attention_definition(q[240:540], k[240:540], v[240:540], decay, [300], dk ** -0.5,
                                     torch.zeros(1, 2, dk, dk, device="cuda"))
    close(o[240:540], ref, TOL[dtype])
    close(left[1:2], want, TOL["f32"])
    assert (o[:40] == 7).all() and (o[650:] == 7).all()  # rows of no sequence stay
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    op.backward(q, k, v, decay, cu, do, *grads, workspace=scratch(op.backward_workspace_bytes(T, 3)))
    x = [t[240:540].double().requires_grad_() for t in (q, k, v)]
    o2, _ = attention_definition(*x, decay, [300], dk ** -0.5, torch.zeros(1, 2, dk, dk, device="cuda"))
    for got, want in zip(grads, torch.autograd.grad((o2 * do[240:540].double()).sum(), x)):
        close(got[240:540], want, TOL[dtype])
        assert (got[:40] == 7).all() and (got[650:] == 7).all()


def test_attention_without_state_slots_and_long_offsets():
    """A slot outside the pool: no state.  Ends past the rows are cut."""
    from tensoroperations_b200 import sequence
    lengths, d = [100, 50, 30], 32
    q, k, v, decay, cu = attention_inputs("f32", lengths, 2, 2, d, d, seed=13)
    op = sequence.LinearAttention("f32", 2, 2, d, d)
    pool = torch.randn(2, 2, d, d, generator=rng(1), device="cuda")
    before = pool.clone()
    slots = torch.tensor([-1, 1, 2], dtype=torch.int32, device="cuda")
    o = torch.empty_like(q)
    cu[3] = 10**6
    op.forward(q, k, v, decay, cu, o, state_in=pool, state_out=pool, slots=slots,
               workspace=scratch(op.workspace_bytes(180, 3)))
    init = torch.zeros(3, 2, d, d, device="cuda")
    init[1] = before[1]
    ref, left = attention_definition(q, k, v, decay, lengths, d ** -0.5, init)
    close(o, ref, TOL["f32"])
    close(pool[1], left[1], TOL["f32"])
    assert torch.equal(pool[0], before[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_in_parts_and_steps(dtype):
    """A prompt in one call, in two calls, and as a prompt with single tokens after it."""
    from tensoroperations_b200 import sequence
    d, T = 64, 330
    q, k, v, decay, cu = attention_inputs(dtype, [T], 4, 2, d, d, seed=14)
    op = sequence.LinearAttention(dtype, 4, 2, d, d)
    ref, left = attention_definition(q, k, v, decay, [T], d ** -0.5, torch.zeros(1, 4, d, d, device="cuda"))
    for first in (1, 128, 201, 320):
        o, S = torch.empty_like(q), torch.zeros(1, 4, d, d, device="cuda")
        for a, b in ((0, first), (first, T)) if first < 320 else ((0, first),):
            op.forward(q[a:b], k[a:b], v[a:b], decay, torch.tensor([0, b - a], dtype=torch.int32, device="cuda"),
                       o[a:b], state_in=S, state_out=S, workspace=scratch(op.workspace_bytes(b - a, 1)))
        if first == 320:
            for t in range(first, T):
                op.step(q[t:t + 1], k[t:t + 1], v[t:t + 1], decay, S, o[t:t + 1])
        close(o, ref, TOL[dtype], f"first {first}")
        close(S, left, TOL["f32"], f"state, first {first}")


@pytest.mark.parametrize("dtype,B,hq,hk,dk,dv", [
    ("bf16", 1, 16, 16, 64, 64), ("bf16", 40, 32, 8, 128, 128), ("f32", 3, 2, 1, 13, 33), ("bf16", 5, 4, 4, 256, 200),
    ("f32", 7, 1, 1, 1, 1), ("f32", 300, 2, 2, 32, 40), ("bf16", 2, 3, 3, 96, 130),
])
def test_attention_step(dtype, B, hq, hk, dk, dv):
    from tensoroperations_b200 import sequence
    q, k, v, decay, _ = attention_inputs(dtype, [B], hq, hk, dk, dv, seed=15)
    pool = torch.randn(B + 2, hq, dk, dv, generator=rng(16), device="cuda")
    slots = torch.randperm(B + 2, generator=rng(17), device="cuda")[:B].to(torch.int32)
    if B > 4:
        slots[2], slots[4] = -1, B + 2  # no state
    before, o = pool.clone(), torch.full((B, hq, dv), float("nan"), dtype=q.dtype, device="cuda")
    op = sequence.LinearAttention(dtype, hq, hk, dk, dv)
    op.step(q, k, v, decay, pool, o, slots=slots)
    want, ref = before.double(), torch.zeros(B, hq, dv, dtype=torch.float64, device="cuda")
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < B + 2:
            y, left = attention_definition(q[r:r + 1], k[r:r + 1], v[r:r + 1], decay, [1], dk ** -0.5, before[s:s + 1])
            ref[r], want[s] = y[0], left[0]
    close(o, ref, TOL[dtype])
    close(pool, want, TOL["f32"])


def test_offsets_past_32_bits():
    """Rows 1.1e9 elements apart and a state at element 2^31 + ..: 64-bit offsets."""
    from tensoroperations_b200 import sequence
    d, far = 64, 1_100_000_000
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GB")
    base = torch.empty(2 * far + 2 * d, dtype=torch.bfloat16, device="cuda")
    q = base.as_strided((3, 2, d), (far, d, 1))
    q.copy_(normal(rng(1), (3, 2, d), "bf16"))
    k, v = normal(rng(2), (3, 2, d), "bf16"), normal(rng(3), (3, 2, d), "bf16")
    decay = torch.tensor([-0.1, -0.01], device="cuda")
    op = sequence.LinearAttention("bf16", 2, 2, d, d)
    o = torch.empty_like(k)
    op.forward(q, k, v, decay, torch.tensor([0, 3], dtype=torch.int32, device="cuda"), o)
    ref, _ = attention_definition(q, k, v, decay, [3], d ** -0.5, torch.zeros(1, 2, d, d, device="cuda"))
    close(o, ref, TOL["bf16"])
    pos = torch.arange(3, dtype=torch.int32, device="cuda").view(1, 3)
    qk = sequence.QkNormRotary("bf16", 2, 2, d)
    yq, yk = torch.empty_like(k), torch.empty_like(k)
    qk.forward(q, k, pos, None, None, yq, yk)
    close(yq, qk_definition(q, None, pos, d, [d // 2], False), TOL["bf16"])
    del base, q
    slots = (1 << 31) // (2 * d * d) + 2
    state = torch.empty(slots, 2, d, d, device="cuda")
    state[-1] = torch.randn(2, d, d, generator=rng(4), device="cuda")
    S = state[-1:].clone()
    at = torch.tensor([slots - 1], dtype=torch.int32, device="cuda")
    q1 = normal(rng(5), (1, 2, d), "bf16")
    op.step(q1, k[:1], v[:1], decay, state, o[:1], slots=at)
    ref, left = attention_definition(q1, k[:1], v[:1], decay, [1], d ** -0.5, S)
    close(o[:1], ref, TOL["bf16"])
    close(state[-1:], left, TOL["f32"])


def test_runs_on_the_stream_it_is_given():
    from tensoroperations_b200 import sequence
    side = torch.cuda.Stream()
    d = 64
    q, k, v, decay, cu = attention_inputs("bf16", [500], 4, 4, d, d, seed=18)
    ref, _ = attention_definition(q, k, v, decay, [500], d ** -0.5, torch.zeros(1, 4, d, d, device="cuda"))
    op = sequence.LinearAttention("bf16", 4, 4, d, d)
    o, ws = torch.zeros_like(q), scratch(op.workspace_bytes(500, 1))
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):  # a launch on any other stream would end the capture
        op.forward(q, k, v, decay, cu, o, workspace=ws, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (o == 0).all()
    graph.replay()
    torch.cuda.synchronize()
    close(o, ref, TOL["bf16"])


def test_refusals_on_the_device():
    from tensoroperations_b200 import sequence
    d = 64
    q, k, v, decay, cu = attention_inputs("bf16", [1000], 4, 2, d, d)
    op = sequence.LinearAttention("bf16", 4, 2, d, d)
    o = torch.full_like(q, 7.0)
    ws = scratch(op.workspace_bytes(1000, 1))
    ok = dict(q=q, k=k, v=v, log_decay=decay, cu_seqlens=cu, o=o, workspace=ws)
    S = torch.zeros(1, 4, d, d, device="cuda")
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(k=k[:10]), dict(v=v.transpose(1, 2)),
                dict(o=o.cpu()), dict(log_decay=decay.double()), dict(cu_seqlens=cu.long()),
                dict(state_in=S[..., :10]), dict(state_out=S.double()), dict(state_in=torch.cat((S, S))),
                dict(slots=torch.zeros(2, dtype=torch.int32, device="cuda"), state_in=S),
                dict(k=k.permute(2, 1, 0).contiguous().permute(2, 1, 0))):
        with pytest.raises(ValueError):
            op.forward(**{**ok, **bad})
    if ws is not None:
        with pytest.raises(ValueError):
            op.forward(**{**ok, "workspace": None})
        with pytest.raises(abi.ToError) as e:
            op.forward(**{**ok, "workspace": ws[:-256]})
        assert e.value.status == abi.TO_ERR_INVALID_ARGUMENT
        with pytest.raises(abi.ToError) as e:
            op.forward(**{**ok, "workspace": torch.empty(ws.numel() + 256, dtype=torch.uint8, device="cuda")[1:]})
        assert e.value.status == abi.TO_ERR_ALIGNMENT
    wide = torch.empty(4 * d * d + 1, device="cuda")[1:].view(1, 4, d, d)
    with pytest.raises(abi.ToError) as e:
        op.forward(**ok, state_out=wide)
    assert e.value.status == abi.TO_ERR_ALIGNMENT
    with pytest.raises(abi.ToError):  # rows that overlap
        op.forward(**{**ok, "k": k[:1].expand(1000, 2, d)})
    torch.cuda.synchronize()
    assert (o == 7).all()  # nothing was launched
