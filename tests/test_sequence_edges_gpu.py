"""The sequence operators at the edges of their ranges, against definitions in float64:
heads split over warps, rows without a length, rows of no sequence, sequences that end in
silence, first tokens, infinities and NaN, streams, autograd.

Tolerances are those of test_sequence_gpu (derived there from the types alone) unless a
test says otherwise.
"""
import math

import pytest

from test_sequence_gpu import (TOL, attention_definition, attention_inputs, close, normal, qk_definition, qk_inputs,
                               rng, scratch)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# ---- query / key norm with rotation ------------------------------------------------


def check_qk_forward(dtype, T, hq, hk, D, inter=False, in_place=False):
    from tensoroperations_b200 import sequence
    q, k, pos, wq, wk = qk_inputs(dtype, T, hq, hk, D, 1, seed=T)
    want = [qk_definition(x, w, pos, D, [D // 2], inter) for x, w in ((q, wq), (k, wk))]
    op = sequence.QkNormRotary(dtype, hq, hk, D, interleaved=inter)
    out = (q, k) if in_place else (torch.full_like(q, float("nan")), torch.full_like(k, float("nan")))
    op.forward(q, k, pos, wq, wk, *out)
    for got, ref, name in zip(out, want, "qk"):
        for h in range(ref.shape[1]):  # head by head: a lost one is a small part of the whole
            close(got[:, h], ref[:, h], TOL[dtype], f"{name} head {h} of {T} tokens")


@pytest.mark.parametrize("dtype,T,hq,hk,D,in_place", [
    ("bf16", 1024, 64, 16, 128, False), ("bf16", 1024, 64, 16, 128, True), ("bf16", 1183, 36, 12, 128, False),
    ("f32", 1100, 16, 4, 256, False), ("f32", 600, 12, 6, 128, True), ("bf16", 900, 30, 10, 64, False),
])
def test_qk_heads_split_over_warps(dtype, T, hq, hk, D, in_place):
    """Tokens too few for the device's warps, heads too many for one warp, several parts of
    tokens for each warp."""
    check_qk_forward(dtype, T, hq, hk, D, in_place=in_place)


@pytest.mark.parametrize("dtype,hq,hk,D,inter", [("bf16", 32, 8, 128, False), ("f32", 24, 3, 96, True)])
def test_qk_heads_at_every_count_of_tokens(dtype, hq, hk, D, inter):
    for T in list(range(300, 2400, 149)) + [1183, 1184, 1185, 2368, 2369]:
        check_qk_forward(dtype, T, hq, hk, D, inter)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,D", [(1, 1, 128), (3, 1, 128), (5, 2, 64), (1, 3, 256), (7, 1, 6)])
def test_qk_gradients_without_eps(dtype, hq, hk, D):
    """eps = 0, no row is zero: the gradients are finite, whatever heads a warp has left over."""
    from tensoroperations_b200 import sequence
    T, half = 41, [D // 2]
    q, k, pos, wq, wk = qk_inputs(dtype, T, hq, hk, D, 1, seed=8)
    g = rng(9)
    gq, gk = normal(g, (T, hq, D), dtype), normal(g, (T, hk, D), dtype)
    op = sequence.QkNormRotary(dtype, hq, hk, D, eps=0.0)
    dq, dk, dwq, dwk = torch.empty_like(gq), torch.empty_like(gk), torch.empty_like(wq), torch.empty_like(wk)
    ws = torch.empty(op.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    op.backward(q, k, pos, wq, wk, gq, gk, dq, dk, dwq, dwk, ws)
    for x, w, gy, dx, dw, name in ((q, wq, gq, dq, dwq, "q"), (k, wk, gk, dk, dwk, "k")):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y = qk_definition(x64, w64, pos, D, half, False, eps=0.0)
        rx, rw = torch.autograd.grad((y * gy.double()).sum(), (x64, w64))
        close(dx, rx, TOL[dtype], "d" + name)
        close(dw, rw, TOL["f32"] * 2, "dw" + name)


# ---- linear attention ----------------------------------------------------------------


@pytest.mark.parametrize("dtype,hq,hk,dk,dv", [
    ("f32", 2, 1, 64, 64), ("bf16", 4, 2, 128, 128), ("bf16", 6, 2, 64, 96), ("bf16", 2, 1, 13, 9)])
def test_gradients_of_shared_heads_leave_rows_of_no_sequence(dtype, hq, hk, dk, dv):
    """Padding before the first sequence and after the last one keeps its gradients, as it does
    where no heads are shared, and whatever the workspace held."""
    from tensoroperations_b200 import sequence
    T, first, last = 700, 40, 650
    q, k, v, decay, _ = attention_inputs(dtype, [T], hq, hk, dk, dv, seed=11)
    do = normal(rng(12), (T, hq, dv), dtype)
    op = sequence.LinearAttention(dtype, hq, hk, dk, dv)
    grads = [torch.full(t.shape, 7.0, dtype=t.dtype, device="cuda") for t in (q, k, v)]
    cu = torch.tensor([first, 240, 240, last], dtype=torch.int32, device="cuda")
    op.backward(q, k, v, decay, cu, do, *grads, workspace=scratch(op.backward_workspace_bytes(T, 3)))
    x = [t[first:last].double().requires_grad_() for t in (q, k, v)]
    o, _ = attention_definition(*x, decay, [200, 0, 410], dk ** -0.5, torch.zeros(3, hq, dk, dv, device="cuda"))
    ref = torch.autograd.grad((o * do[first:last].double()).sum(), x)
    for got, want, name in zip(grads, ref, ("dq", "dk", "dv")):
        close(got[first:last], want, TOL[dtype], name)
        assert (got[:first] == 7).all() and (got[last:] == 7).all(), name
    # and with no sequence that has tokens: nothing is written
    grads = [torch.full(t.shape, 7.0, dtype=t.dtype, device="cuda") for t in (q, k, v)]
    op.backward(q, k, v, decay, torch.full_like(cu, 77), do, *grads,
                workspace=scratch(op.backward_workspace_bytes(T, 3)))
    assert all((g == 7).all() for g in grads)


def packed(T, parts, dtype, by_head):
    """Views of one buffer: each token's parts one after the other, or each head's (all of one head count)."""
    if by_head:
        rows = torch.empty(T, parts[0][0], sum(w for _, w in parts), dtype=dtype, device="cuda")
        return rows.split([w for _, w in parts], -1)
    rows = torch.empty(T, sum(h * w for h, w in parts), dtype=dtype, device="cuda")
    return [x.view(T, *p) for x, p in zip(rows.split([h * w for h, w in parts], -1), parts)]


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("dtype,hq,hk,dk,dv", [("bf16", 4, 4, 64, 128), ("f32", 3, 3, 24, 40), ("bf16", 4, 2, 64, 64)])
def test_packed_rows_hold_inputs_and_outputs(dtype, hq, hk, dk, dv, by_head):
    """Inputs and outputs side by side in the same packed rows share no memory, and are not refused."""
    from tensoroperations_b200 import sequence
    if by_head and hq != hk:
        pytest.skip("heads of one count")
    T, lengths = 390, [300, 90]
    q, k, v, decay, cu = attention_inputs(dtype, lengths, hq, hk, dk, dv, seed=51)
    do = normal(rng(52), (T, hq, dv), dtype)
    parts = [(hq, dk), (hk, dk), (hk, dv), (hq, dv)]
    views = packed(T, parts + parts[:3] + [parts[3]], q.dtype, by_head)
    for view, x in zip(views, (q, k, v, do)):
        view.copy_(x)
    (q1, k1, v1, do1), (dq, dk_, dv_, o) = views[:4], views[4:]
    op = sequence.LinearAttention(dtype, hq, hk, dk, dv)
    op.forward(q1, k1, v1, decay, cu, o, workspace=scratch(op.workspace_bytes(T, 2)))
    op.backward(q1, k1, v1, decay, cu, do1, dq, dk_, dv_, workspace=scratch(op.backward_workspace_bytes(T, 2)))
    x = [t.double().requires_grad_() for t in (q, k, v)]
    ref, _ = attention_definition(*x, decay, lengths, dk ** -0.5, torch.zeros(2, hq, dk, dv, device="cuda"))
    close(o, ref.detach(), TOL[dtype], "o")
    for got, want in zip((dq, dk_, dv_), torch.autograd.grad((ref * do.double()).sum(), x)):
        close(got, want, TOL[dtype], "gradient")
    for view, t in zip(views, (q, k, v, do)):
        assert torch.equal(view, t)
    state = torch.zeros(T, hq, dk, dv, device="cuda")
    op.step(q1, k1, v1, decay, state, o)
    group = hq // hk
    kd, vd = k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    close(o, dk ** -0.5 * (q.double() * kd).sum(-1, keepdim=True) * vd, TOL[dtype], "step")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_qk_in_place_in_packed_rows(dtype):
    from tensoroperations_b200 import sequence
    T, hq, hk, D = 77, 5, 3, 64
    q, k, pos, wq, wk = qk_inputs(dtype, T, hq, hk, D, 1, seed=53)
    gq, gk = (normal(rng(54 + i), x.shape, dtype) for i, x in enumerate((q, k)))
    op = sequence.QkNormRotary(dtype, hq, hk, D)
    ws = torch.empty(op.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    dq, dk, dw = torch.empty_like(gq), torch.empty_like(gk), torch.empty(2, D, device="cuda")
    op.backward(q, k, pos, wq, wk, gq, gk, dq, dk, dw[0], dw[1], ws)
    q2, k2, _, _, _ = qk_inputs(dtype, T, hq, hk, D, 1, seed=53)  # the gradients over the inputs
    op.backward(q2, k2, pos, wq, wk, gq, gk, q2, k2, None, None, ws)
    assert torch.equal(q2, dq) and torch.equal(k2, dk)
    want = [qk_definition(x, w, pos, D, [D // 2], False) for x, w in ((q, wq), (k, wk))]
    op.forward(q, k, pos, wq, wk, q, k)
    close(q, want[0], TOL[dtype], "q")
    close(k, want[1], TOL[dtype], "k")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,silent,rates", [(300, 172, [-0.04, -0.06, -0.09]), (6000, 1500, [-0.004, -0.006, -0.008])])
def test_states_of_sequences_that_end_in_silence(dtype, T, silent, rates):
    """Tokens of zero keys at the end (zero outputs' gradients at the beginning, for the state's
    gradient): what is left of the others has decayed far, and is still exact to f32."""
    from tensoroperations_b200 import sequence
    d, H = 64, 3
    q, k, v, _, cu = attention_inputs(dtype, [T], H, H, d, d, seed=21)
    decay = torch.tensor(rates, device="cuda")
    do = normal(rng(22), (T, H, d), dtype)
    k[T - silent:] = 0
    do[:silent] = 0
    op = sequence.LinearAttention(dtype, H, H, d, d)
    o, left, dS = torch.empty_like(q), torch.empty(1, H, d, d, device="cuda"), torch.empty(1, H, d, d, device="cuda")
    op.forward(q, k, v, decay, cu, o, state_out=left, workspace=scratch(op.workspace_bytes(T, 1)))
    grads = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, v)]
    op.backward(q, k, v, decay, cu, do, *grads, dstate_in=dS, workspace=scratch(op.backward_workspace_bytes(T, 1)))
    lam = decay.double()
    age = torch.arange(T, device="cuda", dtype=torch.float64)
    for h in range(H):
        late = (lam[h] * (T - 1 - age)).exp()[:, None]
        close(left[0, h], (k[:, h].double() * late).t() @ v[:, h].double(), TOL["f32"], f"state, head {h}")
        early = d ** -0.5 * (lam[h] * (age + 1)).exp()[:, None]
        close(dS[0, h], (q[:, h].double() * early).t() @ do[:, h].double(), TOL["f32"], f"dstate, head {h}")


def rounded_once(got, ref, what):
    """Half the spacing of bf16 values (2^-7 of the power of two below), and what two planes leave of P."""
    half = 0.5 * 2.0 ** (ref.abs().clamp(min=1e-30).log2().floor() - 7)
    off = ((got.double() - ref).abs() - half) / ref.abs().amax(-1, True)
    assert (off <= 2.0 ** -14).all(), (what, float(off.max()))


@pytest.mark.parametrize("tokens", [31, 32, 33, 48, 100, 128, 129, 400])
def test_first_tokens_do_not_depend_on_how_many_follow(tokens):
    """The first tokens of a sequence (the last ones, for dk and dv) have the result's own rounding
    alone, however long the sequence is."""
    from tensoroperations_b200 import sequence
    H, d, n = 4, 128, min(tokens, 32)
    q, k, v, decay, cu = attention_inputs("bf16", [tokens], H, H, d, 64, seed=31)
    op = sequence.LinearAttention("bf16", H, H, d, 64)
    o = torch.empty(tokens, H, 64, dtype=q.dtype, device="cuda")
    op.forward(q, k, v, decay, cu, o, workspace=scratch(op.workspace_bytes(tokens, 1)))
    none = torch.zeros(1, H, d, 64, device="cuda")
    x = [t.double().requires_grad_() for t in (q, k, v)]
    ref, _ = attention_definition(*x, decay, [tokens], d ** -0.5, none)
    rounded_once(o[:n], ref.detach()[:n], "o")
    do = normal(rng(32), (tokens, H, 64), "bf16")
    grads = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, v)]
    op.backward(q, k, v, decay, cu, do, *grads, workspace=scratch(op.backward_workspace_bytes(tokens, 1)))
    dq, dk, dv = torch.autograd.grad((ref * do.double()).sum(), x)
    rounded_once(grads[0][:n], dq[:n], "dq")
    rounded_once(grads[1][tokens - n:], dk[tokens - n:], "dk")
    rounded_once(grads[2][tokens - n:], dv[tokens - n:], "dv")


# tokens j of the poisoned rows: inside chunks of 64 and 128, at their ends, in a later sequence's first chunk
POISON = [("f32", 64, 48), ("f32", 130, 72), ("bf16", 40, 13), ("bf16", 136, 24),
          ("bf16", 128, 128), ("bf16", 64, 80), ("bf16", 40, 16)]
SPOTS = [(0,), (63,), (64, 200), (100,), (127,), (128, 131), (255,), (299,)]


def poisoned(t, spots, head, col, value):
    """t with `value` at (spot, head, col), and t with zeros there."""
    bad, clean = t.clone(), t.clone()
    for s in spots:
        bad[s, head, col], clean[s, head, col] = value, 0
    return bad, clean


def attention_sums(q, k, v, decay, lengths, scale):
    """o as sums over the earlier tokens, in float64 (each head its own key and value head)."""
    out, first = [], 0
    for n in lengths:
        a, b, c = (t[first:first + n].double().transpose(0, 1) for t in (q, k, v))
        i = torch.arange(n, device="cuda", dtype=torch.float64)
        gap = i[:, None] - i
        weigh = torch.where(gap >= 0, (decay.double()[:, None, None] * gap.clamp(min=0)).exp(), 0.0)
        out.append((scale * ((a @ b.transpose(1, 2)) * weigh) @ c).transpose(0, 1))
        first += n
    return torch.cat(out)


def check_spread(got, ref, hit, dtype, what):
    """`hit`: what depends on a poisoned value.  It is not finite, everything else is right."""
    fin = torch.isfinite(got)
    assert (fin == ~hit).all(), (what, "lost", int((~fin & ~hit).sum()), "kept", int((fin & hit).sum()))
    close(torch.where(hit, torch.zeros_like(got), got), torch.where(hit, torch.zeros_like(ref), ref), TOL[dtype], what)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype,dk,dv", POISON)
def test_non_finite_values_do_not_go_back_in_time(dtype, dk, dv, value):
    """An infinite or NaN query, key or value makes what depends on it non-finite, and nothing else."""
    from tensoroperations_b200 import sequence
    lengths, H, scale = [300, 90], 2, 0.2
    T = sum(lengths)
    q, k, v, _, cu = attention_inputs(dtype, lengths, H, H, dk, dv, seed=41)
    decay = torch.tensor([-0.01, -0.3], device="cuda")
    op = sequence.LinearAttention(dtype, H, H, dk, dv, scale=scale)
    t = torch.arange(T, device="cuda")
    none = torch.zeros(2, H, dk, dv, device="cuda")
    for n, spots in enumerate(SPOTS):
        h, c = n % H, (7 * n + 3) % min(dk, dv)
        for name in "qkv":
            x = dict(q=q, k=k, v=v)
            bad, clean = poisoned(x[name], spots, h, c, value)
            ref = attention_sums(**{**x, name: clean}, decay=decay, lengths=lengths, scale=scale)
            o, left = torch.empty(T, H, dv, dtype=q.dtype, device="cuda"), torch.empty_like(none)
            op.forward(**{**x, name: bad}, log_decay=decay, cu_seqlens=cu, o=o, state_out=left,
                       workspace=scratch(op.workspace_bytes(T, 2)))
            hit, shit = torch.zeros(T, H, dv, dtype=torch.bool, device="cuda"), torch.zeros_like(none, dtype=torch.bool)
            after = (t >= spots[0]) & (t < lengths[0])
            if name == "q":
                hit[list(spots), h] = True
            elif name == "k":
                hit[after, h] = True
                shit[0, h, c] = True
            else:
                hit[after, h, c] = True
                shit[0, h, :, c] = True
            check_spread(o, ref, hit, dtype, f"o, {name} at {spots}")
            assert (torch.isfinite(left) == ~shit).all(), (name, spots)


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("dtype,dk,dv", POISON)
def test_non_finite_values_in_gradients(dtype, dk, dv, value):
    """dq sees earlier keys and values, dk and dv later queries and outputs' gradients, no others."""
    from tensoroperations_b200 import sequence
    lengths, H, scale = [300, 90], 2, 0.2
    T = sum(lengths)
    q, k, v, _, cu = attention_inputs(dtype, lengths, H, H, dk, dv, seed=42)
    do = normal(rng(43), (T, H, dv), dtype)
    decay = torch.tensor([-0.01, -0.3], device="cuda")
    op = sequence.LinearAttention(dtype, H, H, dk, dv, scale=scale)
    t = torch.arange(T, device="cuda")
    for n, spots in enumerate(SPOTS):
        h, c = n % H, (7 * n + 3) % min(dk, dv)
        for name in ("q", "k", "v", "do"):
            x = dict(q=q, k=k, v=v, do=do)
            bad, clean = poisoned(x[name], spots, h, c, value)
            y = {m: a.double().requires_grad_() for m, a in {**x, name: clean}.items()}
            ref = attention_sums(y["q"], y["k"], y["v"], decay, lengths, scale)
            refs = torch.autograd.grad((ref * y["do"]).sum(), (y["q"], y["k"], y["v"]))
            grads = [torch.empty(a.shape, dtype=a.dtype, device="cuda") for a in (q, k, v)]
            y = {**x, name: bad}
            op.backward(y["q"], y["k"], y["v"], decay, cu, y["do"], *grads,
                        workspace=scratch(op.backward_workspace_bytes(T, 2)))
            hit = [torch.zeros(a.shape, dtype=torch.bool, device="cuda") for a in (q, k, v)]
            after, upto, at = (t >= spots[0]) & (t < lengths[0]), t <= spots[-1], list(spots)
            if name == "q":
                hit[1][upto, h, c] = True
                hit[2][upto, h] = True
            elif name == "k":
                hit[0][after, h, c] = True
                hit[2][at, h] = True
            elif name == "v":
                hit[0][after, h] = True
                hit[1][at, h] = True
            else:
                hit[0][at, h] = True
                hit[1][upto, h] = True
                hit[2][upto, h, c] = True
            for got, want, where, what in zip(grads, refs, hit, ("dq", "dk", "dv")):
                check_spread(got, want, where, dtype, f"{what}, {name} at {spots}")


# ---- streams and autograd ---------------------------------------------------------------


def every_call(stream=None):
    """The five calls on small tensors: (what they write, the call) each; `stream` as in the calls."""
    from tensoroperations_b200 import sequence
    T, H, d = 200, 2, 64
    q, k, v, decay, cu = attention_inputs("bf16", [T], H, H, d, d, seed=61)
    more = {} if stream is None else dict(stream=stream)
    pos = torch.arange(T, dtype=torch.int32, device="cuda").view(1, T)
    qk, la = sequence.QkNormRotary("bf16", H, H, d), sequence.LinearAttention("bf16", H, H, d, d)
    w = [torch.ones(d, device="cuda") for _ in range(4)]
    out = lambda: torch.zeros(T, H, d, dtype=q.dtype, device="cuda")  # noqa: E731
    ws = scratch(max(qk.workspace_bytes(T), la.workspace_bytes(T, 1), la.backward_workspace_bytes(T, 1), 256))
    a, b, c, o, g = out(), out(), out(), out(), normal(rng(62), (T, H, d), "bf16")
    state, left = torch.zeros(T, H, d, d, device="cuda"), torch.zeros(1, H, d, d, device="cuda")
    first, second = out(), out()
    yield (a, b), lambda: qk.forward(q, k, pos, w[0], w[1], a, b, **more)
    yield (first, second, w[2], w[3]), lambda: qk.backward(q, k, pos, w[0], w[1], g, g, first, second, w[2], w[3], ws,
                                                           **more)
    yield (o, left), lambda: la.forward(q, k, v, decay, cu, o, state_out=left, workspace=ws, **more)
    o1 = out()
    yield (o1, state), lambda: la.step(q, k, v, decay, state, o1, **more)
    dq, dk, dS = out(), out(), torch.zeros_like(left)
    yield (dq, dk, c, dS), lambda: la.backward(q, k, v, decay, cu, g, dq, dk, c, dstate_out=left, dstate_in=dS,
                                               workspace=ws, **more)


def test_calls_run_on_the_current_stream():
    """Without a stream a call runs on torch's current one, as what torch does to its tensors."""
    for written, call in every_call():
        before = [t.clone() for t in written]
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):  # (a launch on any other stream is not recorded)
            call()
        torch.cuda.synchronize()
        assert all(torch.equal(t, b) for t, b in zip(written, before))
        graph.replay()
        torch.cuda.synchronize()
        assert not any(torch.equal(t, b) for t, b in zip(written, before))


def test_stream_zero_is_the_default_stream():
    want = []
    for written, call in every_call():
        call()
        want.append([t.clone() for t in written])
    for (written, call), ref in zip(every_call(stream=0), want):
        call()
        torch.cuda.synchronize()
        assert all(torch.equal(t, r) for t, r in zip(written, ref))


# ---- autograd: what is written is known to be


def test_written_tensors_are_known_to_autograd():
    """A tensor that autograd has saved and a call overwrites is an error in the backward pass, not a
    wrong gradient; what a call reads stays as it was."""
    for written, call in every_call():
        x = [torch.ones(t.shape, device="cuda", requires_grad=True) for t in written]
        y = [a * t for a, t in zip(x, written)]  # saves t
        before = [t._version for t in written]
        call()
        assert all(t._version > b for t, b in zip(written, before))
        for out in y:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()
    q, k, v, decay, cu = attention_inputs("bf16", [50], 2, 2, 64, 64)
    from tensoroperations_b200 import sequence
    op, o, S = sequence.LinearAttention("bf16", 2, 2, 64, 64), torch.empty_like(q), torch.zeros(1, 2, 64, 64, device="cuda")
    before = [t._version for t in (q, k, v, decay, cu, S)]
    op.forward(q, k, v, decay, cu, o, state_in=S)
    assert [t._version for t in (q, k, v, decay, cu, S)] == before
    with torch.inference_mode():  # tensors without versions
        op.forward(q, k, v, decay, cu, torch.empty_like(q), state_in=S)
