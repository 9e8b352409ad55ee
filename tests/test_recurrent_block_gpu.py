"""The gated recurrence, the norms around a block and rows in 8 bits against plain 64-bit forms."""
import pytest

torch = pytest.importorskip("torch")
from tensoroperations_b200 import abi, sequence  # noqa: E402
from tests import recurrent_block_oracle as R  # noqa: E402
from tests.recurrent_block_oracle import U, d  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def cuda(*shape, gen, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def close(got, want, tol, what):
    """Everywhere within tol; where `want` is not finite, so is `got`."""
    got, want = d(got), d(want)
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: infinities elsewhere"
    off = torch.where(fine, (got - want).abs(), 0.0) - torch.where(fine, torch.as_tensor(tol).expand_as(want), 0.0)
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max():.3g} over the bound"


# ---- 8 bits --------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,width,offset", [(1, 1, 0), (3, 31, 0), (5, 32, 0), (7, 33, 1), (2, 48, 0), (129, 64, 0),
                                                 (40, 128, 8), (33, 1000, 0), (17, 1237, 3), (600, 512, 0)])
def test_eight_bits(dtype, tokens, width, offset):
    gen = torch.Generator("cuda").manual_seed(tokens * width)
    whole = cuda(tokens, width + 2 * offset, gen=gen) * torch.exp(3 * cuda(width + 2 * offset, gen=gen))
    whole[0, :] *= 1e-37  # scales near the least one
    if tokens > 2:
        whole[1, :] = 0
        whole[2, : width // 2] = 127.0 * 2 ** 5  # exactly at a scale's end
    x = whole.to(dtype)[:, offset:offset + width]
    if tokens > 4 and width > 32:
        x[3, 1] = float("inf")
        x[4, width - 1] = float("nan")
    op = sequence.Checkpoint8(dtype, width)
    x8 = sequence.Rows8.empty(tokens, width)
    op.pack(x, x8)
    codes, scales = R.pack8(x)
    assert torch.equal(x8.codes.cpu(), codes)
    assert torch.equal(x8.scales.cpu(), scales)
    out = torch.empty(tokens, width + 5, dtype=dtype, device="cuda")[:, :width]
    op.unpack(x8, out)
    want = R.unpack8(codes, scales)
    assert torch.equal(d(out).nan_to_num(7.0), want.to(dtype).double().nan_to_num(7.0))
    fine = torch.isfinite(want)
    most = torch.zeros_like(want)
    for k in range(0, width, 32):
        most[:, k:k + 32] = d(x)[:, k:k + 32].abs().amax(1, keepdim=True)
    assert ((want - d(x)).abs()[fine] <= (most / 127 + 2.0 ** -128)[fine]).all()


def test_eight_bits_of_no_rows():
    op = sequence.Checkpoint8("bf16", 40)
    x = torch.empty(0, 40, dtype=BF16, device="cuda")
    op.pack(x, sequence.Rows8.empty(0, 40))
    op.unpack(sequence.Rows8.empty(0, 40), x)


# ---- the recurrence ------------------------------------------------------------------


LENGTHS = [[1], [0], [128], [129], [3, 0, 0, 1, 300, 128, 0], [2500], [5000, 77], [64] * 9, [1] * 40]


def rows(tokens, channels, dtype, gen, layout):
    """x and f: two arrays, or views into packed rows (at odd addresses where the width is odd)."""
    if layout == "apart":
        return cuda(tokens, channels, gen=gen, dtype=dtype), cuda(tokens, channels, gen=gen, dtype=dtype, scale=2.0)
    packed = cuda(tokens, 2 * channels + 3, gen=gen, dtype=dtype)
    return packed[:, 1:1 + channels], packed[:, 1 + channels:1 + 2 * channels]


def recurrence_case(dtype, channels, lengths, complement, layout, keep, bias=True, spare=0, seed=0):
    """Everything of one forward and backward call, checked."""
    gen = torch.Generator("cuda").manual_seed(seed + channels * 7 + sum(lengths))
    n, tokens = len(lengths), sum(lengths) + spare
    x, f = rows(tokens, channels, dtype, gen, layout)
    b = 4 * torch.rand(channels, generator=gen, device="cuda") if bias else None
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    op = sequence.GatedRecurrence(dtype, channels, complement)
    state = cuda(n + 2, channels, gen=gen)
    slots = torch.randperm(n + 2, generator=gen, device="cuda")[:n].to(torch.int32)
    entered = state.clone()
    h = torch.full((tokens, channels), 7.0, dtype=dtype, device="cuda")
    saved = torch.empty(op.saved_rows(tokens, n), channels, device="cuda")
    ws = torch.full((max(op.workspace_bytes(tokens, n), 1),), 255, dtype=torch.uint8, device="cuda")
    kept = {}
    if keep:
        kept = {"keep_" + k: sequence.Rows8.empty(tokens, channels) for k in "xf"}
    op.forward(x, f, b, cu, h, state_in=state, state_out=state, slots=slots, saved=saved, workspace=ws, **kept)
    assert abi.lib.to_device_status(1) == 0
    bd = None if b is None else d(b)
    x0, f0, s0 = d(x), d(f), d(entered)[slots.cpu().long()]
    want, before, left, a, z = R.recurrence(x0, f0, bd, lengths, s0, complement)
    used = sum(lengths)
    size = torch.cat((want[:used], s0, x0[:used] if complement else x0[:0], before[:used])).abs().amax(0)
    g0 = f0 if b is None else f0 + bd
    bound = R.chain_bound(z, g0, size)
    close(h[:used], want[:used], bound + R.rounding(dtype) * want[:used].abs(), "h")
    assert (h[used:] == 7.0).all()
    close(state[slots.long()], left, bound, "state")
    other = torch.ones(n + 2, dtype=torch.bool, device="cuda")
    other[slots.long()] = False
    assert torch.equal(state[other], entered[other])
    if keep:
        for k, t in (("keep_x", x), ("keep_f", f)):
            codes, scales = R.pack8(t)
            assert torch.equal(kept[k].codes[:used].cpu(), codes[:used]), k
            assert torch.equal(kept[k].scales[:used].cpu(), scales[:used]), k
        # from the forward pass's states at the head of every segment on
        x0, f0 = (R.unpack8(*R.pack8(t)) for t in (x, f))
        pieces = [min(R.SEGMENT, m - i) for m in lengths for i in range(0, m, R.SEGMENT)]
        heads = torch.tensor([0] + pieces).cumsum(0)[:-1]
        _, before, _, a, z = R.recurrence(x0, f0, bd, pieces, before[heads], complement)
        before = torch.cat((before[:used], before.new_full((spare, channels), torch.nan)))
    dh = cuda(tokens, channels, gen=gen, dtype=dtype)
    dstate = cuda(n, channels, gen=gen)
    dx, df = (torch.full((tokens, channels), 7.0, dtype=dtype, device="cuda") for _ in "xf")
    dbias, into = torch.full((channels,), 7.0, device="cuda"), torch.full((n, channels), 7.0, device="cuda")
    ws = torch.full((max(op.backward_workspace_bytes(tokens, n), 1),), 255, dtype=torch.uint8, device="cuda")
    op.backward(kept.get("keep_x", x), kept.get("keep_f", f), b, cu, saved, dh, dx, df, dbias, dstate_out=dstate,
                dstate_in=into, workspace=ws)
    assert abi.lib.to_device_status(1) == 0
    wx, wf, wb, ws_, G = R.recurrence_grad(x0, a, z, before, lengths, d(dh), d(dstate), complement)
    gsize = torch.cat((G[:used], d(dh)[:used], d(dstate))).abs().amax(0)
    g0 = f0 if b is None else f0 + bd
    gb = R.chain_bound(z, g0, gsize)
    hb = R.chain_bound(z, g0, torch.cat((size[None], before[:used].abs(), x0[:used].abs())).amax(0))
    gate = U * (2 * g0.abs() + 16)  # of z and of a z, relative
    e = before - x0 if complement else before
    tx = (z * gb + gate * (z * G).abs() if complement else gb)[:used]
    close(dx[:used], wx[:used], tx + R.rounding(dtype) * wx[:used].abs(), "dx")
    tf = ((a * z) * (gb * e.abs() + G.abs() * (hb + 4 * U * size)) + (gate + 8 * U) * wf.abs())[:used]
    close(df[:used], wf[:used], tf + R.rounding(dtype) * wf[:used].abs(), "df")
    assert (dx[used:] == 7.0).all() and (df[used:] == 7.0).all()
    close(dbias, wb, tf.sum(0) + 32 * U * wf[:used].abs().sum(0) + U * wb.abs(), "dbias")
    close(into, ws_, gb + U * ws_.abs(), "dstate_in")


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "x".join(map(str, v[:5])))
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("keep", [False, True])
def test_recurrence_lengths(lengths, dtype, keep):
    recurrence_case(dtype, 96, lengths, True, "apart", keep)


@pytest.mark.parametrize("channels", [1, 2, 31, 33, 64, 65, 130, 319])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("keep", [False, True])
def test_recurrence_channels(channels, dtype, keep):
    recurrence_case(dtype, channels, [3, 0, 200, 1, 129], channels % 2 == 0, "packed", keep, bias=channels != 2, spare=5)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_recurrence_plain_input(dtype):
    recurrence_case(dtype, 72, [700, 5, 300], False, "apart", True, spare=200)


def test_recurrence_many_segments():
    recurrence_case(F32, 40, [9000], True, "apart", False)


def test_recurrence_without_states_and_single_segments():
    """Calls of at most 64 tokens need no workspace; no states, no gradients of bias and states."""
    op = sequence.GatedRecurrence("f32", 50)
    assert op.workspace_bytes(64, 4) == 0
    gen = torch.Generator("cuda").manual_seed(1)
    x, f, dh = (cuda(64, 50, gen=gen) for _ in range(3))
    cu = torch.tensor([0, 50, 50, 64], dtype=torch.int32, device="cuda")
    h, dx, df = (torch.empty_like(x) for _ in range(3))
    saved = torch.empty(op.saved_rows(64, 3), 50, device="cuda")
    op.forward(x, f, None, cu, h, saved=saved)
    ws = torch.empty(op.backward_workspace_bytes(64, 3), dtype=torch.uint8, device="cuda")
    op.backward(x, f, None, cu, saved, dh, dx, df, workspace=ws)
    zero = torch.zeros(3, 50, dtype=torch.float64)
    want, before, _, a, z = R.recurrence(d(x), d(f), None, [50, 0, 14], zero, True)
    wx, wf, *_ = R.recurrence_grad(d(x), a, z, before, [50, 0, 14], d(dh), zero, True)
    close(h, want, R.chain_bound(z, d(f), d(x).abs().amax(0)), "h")
    g = R.chain_bound(z, d(f), 50 * d(dh).abs().amax(0))
    close(dx, wx, g, "dx")
    close(df, wf, 20 * g, "df")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("requests,channels,complement", [(1, 1, True), (3, 64, False), (40, 130, True), (5, 1024, True)])
def test_step(dtype, requests, channels, complement):
    gen = torch.Generator("cuda").manual_seed(requests)
    x, f = rows(requests, channels, dtype, gen, "apart" if channels % 4 == 0 else "packed")
    bias = cuda(channels, gen=gen, scale=3.0)
    state = cuda(requests + 2, channels, gen=gen)
    entered = state.clone()
    slots = torch.randperm(requests + 2, generator=gen, device="cuda")[:requests].to(torch.int32)
    slots[0] = requests + 2 if requests > 1 else slots[0]  # outside: no state
    h = torch.empty(requests, channels, dtype=dtype, device="cuda")
    op = sequence.GatedRecurrence(dtype, channels, complement)
    op.step(x, f, bias, state, h, slots=slots)
    for i in range(requests):
        at = int(slots[i])
        if at >= requests + 2:
            assert (h[i] == 0).all()
            continue
        want, _, left, _, z = R.recurrence(d(x)[i:i + 1], d(f)[i:i + 1], d(bias), [1], d(entered)[at:at + 1], complement)
        size = torch.stack((want[0].abs(), d(x)[i].abs(), d(entered)[at].abs())).amax(0)
        bound = R.chain_bound(z, d(f)[i:i + 1] + d(bias), size)
        close(state[at:at + 1], left, bound, "state")
        close(h[i:i + 1], want, bound + R.rounding(dtype) * want.abs(), "h")


def test_step_follows_prompt():
    """A sequence as one prompt, and as a prompt with single tokens after it."""
    gen = torch.Generator("cuda").manual_seed(3)
    x, f = cuda(260, 96, gen=gen), cuda(260, 96, gen=gen, scale=2.0)
    op = sequence.GatedRecurrence("f32", 96)
    ws = torch.empty(op.workspace_bytes(260, 1), dtype=torch.uint8, device="cuda")

    def prompt(n, state):
        h = torch.empty(n, 96, device="cuda")
        op.forward(x[:n], f[:n], None, torch.tensor([0, n], dtype=torch.int32, device="cuda"), h, state_out=state, workspace=ws)
        return h

    state = torch.empty(1, 96, device="cuda")
    whole = prompt(260, torch.empty(1, 96, device="cuda"))
    prompt(250, state)
    out = []
    for i in range(250, 260):
        h = torch.empty(1, 96, device="cuda")
        op.step(x[i:i + 1], f[i:i + 1], None, state, h)
        out.append(h)
    z = torch.sigmoid(-d(f))
    close(torch.cat(out), whole[250:], 2 * R.chain_bound(z, d(f), d(x).abs().amax(0)), "h")


# ---- the norms -----------------------------------------------------------------------


def norm_case(dtype, residual, width, tokens, gate, keep=False, post_norm=True, weights=True, layout="apart", scale=0.7,
              eps=1e-6, skip=True, grad_n=True):
    gen = torch.Generator("cuda").manual_seed(width * 3 + tokens)
    pad = 0 if layout == "apart" else 3

    def make(kind, s=1.0):
        return cuda(tokens, width + pad, gen=gen, dtype=kind, scale=s)[:, :width]

    r, y, g = make(residual, 2.0), make(dtype), make(dtype, 3.0) if gate else None
    wp, wn = (1 + 0.3 * cuda(width, gen=gen) for _ in "ab") if weights else (None, None)
    op = sequence.BlockNorm(dtype, width, residual=residual, gate=gate, post_norm=post_norm, scale=scale, eps=eps)
    ro, n = make(residual), make(dtype)
    kept = {k: sequence.Rows8.empty(tokens, width) for k in ("keep_r", "keep_y", "keep_g")[:3 if gate else 2]} if keep else {}
    op.forward(r, y, g, wp, wn, ro, n, **kept)
    ones = torch.ones(width, dtype=torch.float64)
    p0, n0 = (ones, ones) if wp is None else (d(wp), d(wn))
    r0, y0 = d(r), d(y)
    a0, _ = R.act(gate, d(g)) if gate else (torch.ones_like(y0), None)
    py = R.rms(y0, eps) if post_norm else torch.ones(tokens, 1, dtype=torch.float64)
    v = scale * p0 * y0 / py * a0
    # sums of `width` squares and the root: 32 additions in a row at most, halved by the root; the products,
    # and the gate's exp (|g| U) and quotient
    count = 64 * U
    gate_off = U * (2 * d(g).abs() + 16) if gate else torch.zeros_like(y0)
    want = r0 + v
    tr = 2 * U * (r0.abs() + v.abs()) + (count + gate_off) * v.abs()
    close(ro, want, tr + R.rounding(residual) * want.abs(), "r_out")
    size = R.rms(want, eps)
    wantn = n0 * want / size
    mean = (want.abs() * tr).mean(-1, keepdim=True) / size.square()  # the sum's share of tr, relative
    tn = n0.abs() * tr / size + (count + mean) * wantn.abs()
    close(n, wantn, tn + R.rounding(dtype) * wantn.abs(), "n")
    if keep:
        # r_out before its rounding: within a step of the group's scale, the inputs exactly
        for k, t in (("keep_y", y), ("keep_g", g))[:2 if gate else 1]:
            codes, scales = R.pack8(t)
            assert torch.equal(kept[k].codes.cpu(), codes) and torch.equal(kept[k].scales.cpu(), scales), k
        most = torch.zeros_like(want)
        for k in range(0, width, 32):
            most[:, k:k + 32] = want[:, k:k + 32].abs().amax(1, keepdim=True)
        close(R.unpack8(*kept["keep_r"]), want, most / 127 + 2 * tr + 64 * U * most, "keep_r")
    # gradients from the values given
    dro, dn = make(residual) if skip else None, make(dtype) if grad_n else None
    dr, dy, dg = make(residual), make(dtype), make(dtype) if gate else None
    dwp, dwn = (torch.full((width,), 7.0, device="cuda") for _ in "ab")
    ws = torch.full((op.workspace_bytes(tokens),), 255, dtype=torch.uint8, device="cuda")
    op.backward(kept.get("keep_r", ro), kept.get("keep_y", y), kept.get("keep_g", g), wp, wn, dro, dn, dr, dy, dg, dwp, dwn, ws)
    val = lambda t, k: R.unpack8(*kept[k]) if k in kept else d(t)  # noqa: E731
    r0, y0 = val(ro, "keep_r"), val(y, "keep_y")
    a0, slope = R.act(gate, val(g, "keep_g")) if gate else (torch.ones_like(y0), torch.zeros_like(y0))
    py = R.rms(y0, eps) if post_norm else torch.ones(tokens, 1, dtype=torch.float64)
    zero = torch.zeros_like(r0)
    s0, dn0 = zero if dro is None else d(dro), zero if dn is None else d(dn)
    pr = R.rms(r0, eps)
    e, rh = n0 * dn0, r0 / pr
    back = rh * (e * rh).mean(-1, keepdim=True) / pr
    t = s0 + e / pr - back
    sums = rh.abs() * (e * rh).abs().mean(-1, keepdim=True) / pr
    tt = 2 * count * (e.abs() / pr + sums) + 4 * U * s0.abs()
    close(dr, t, tt + R.rounding(residual) * t.abs(), "dr")
    q, yh = scale * t, y0 / py
    tq = abs(scale) * tt
    close(dwn, (dn0 * rh).sum(0), (tokens + 64) * U * (dn0 * rh).abs().sum(0), "dw_pre")
    if gate:
        wg = q * p0 * yh * slope
        # (silu's slope p + g p q may cancel: its parts count)
        g0 = val(g, "keep_g")
        parts = torch.sigmoid(g0) * (1 + g0.abs()) if gate == "silu" else slope.abs()
        tg = (p0 * yh).abs() * (tq * slope.abs() + q.abs() * parts * (count + gate_off))
        close(dg, wg, tg + R.rounding(dtype) * wg.abs(), "dg")
    du = q * a0
    tu = (tq + q.abs() * (count + gate_off)) * a0.abs()
    close(dwp, (du * yh).sum(0), ((tokens + 64) * U * (du * yh).abs() + tu * yh.abs()).sum(0), "dw_post")
    e = p0 * du
    te = p0.abs() * tu
    if post_norm:
        wy = (e - yh * (e * yh).mean(-1, keepdim=True)) / py
        ty = (te + yh.abs() * ((te + 2 * count * e.abs()) * yh.abs()).mean(-1, keepdim=True)) / py + \
            2 * count * (e.abs() + yh.abs() * (e * yh).abs().mean(-1, keepdim=True)) / py
    else:
        wy, ty = e, te + count * e.abs()
    close(dy, wy, ty + R.rounding(dtype) * wy.abs(), "dy")


@pytest.mark.parametrize("width", [1, 7, 8, 40, 256, 257, 264, 1000, 1003, 2048, 4096, 8200, 16384])
@pytest.mark.parametrize("dtype,residual", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_norm_widths(width, dtype, residual):
    norm_case(dtype, residual, width, 5 if width > 2048 else 37, "silu")


@pytest.mark.parametrize("gate", [None, "linear", "sigmoid", "silu"])
@pytest.mark.parametrize("width", [72, 100, 333, 512])
@pytest.mark.parametrize("dtype,residual", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_norm_kept(gate, width, dtype, residual):
    norm_case(dtype, residual, width, 19, gate, keep=True, layout="apart" if width % 8 == 0 else "packed")


@pytest.mark.parametrize("more", [dict(post_norm=False), dict(weights=False), dict(skip=False), dict(grad_n=False),
                                  dict(scale=-2.0), dict(scale=0.0), dict(layout="packed"), dict(eps=0.0),
                                  dict(tokens=1), dict(tokens=700)], ids=str)
def test_norm_options(more):
    for dtype, residual in ((BF16, F32), (F32, F32)):
        norm_case(dtype, residual, **{**dict(width=136, tokens=33, gate="sigmoid"), **more})


@pytest.mark.parametrize("width", [136, 133])
def test_norm_alone(width):
    """A model's first norm: no block, no residual sum; and the last sum, which no norm follows."""
    gen = torch.Generator("cuda").manual_seed(width)
    r, w = cuda(30, width, gen=gen), 1 + 0.3 * cuda(width, gen=gen)
    op = sequence.BlockNorm("bf16", width, residual="f32", gate="silu")
    n = torch.empty(30, width, dtype=BF16, device="cuda")
    kept = sequence.Rows8.empty(30, width)
    op.forward(r, None, None, None, w, None, n, keep_r=kept)
    codes, scales = R.pack8(r)
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)
    size = R.rms(d(r), 1e-6)
    want = d(w) * d(r) / size
    close(n, want, (R.half(BF16) + 64 * U) * want.abs(), "n")
    dn, dro = cuda(30, width, gen=gen, dtype=BF16), cuda(30, width, gen=gen)
    dr, dw = torch.empty_like(r), torch.empty(width, device="cuda")
    ws = torch.empty(op.workspace_bytes(30), dtype=torch.uint8, device="cuda")
    op.backward(r, None, None, None, w, dro, dn, dr, None, None, None, dw, ws)
    e, rh = d(w) * d(dn), d(r) / size
    want = d(dro) + (e - rh * (e * rh).mean(-1, keepdim=True)) / size
    close(dr, want, 128 * U * ((e.abs() + rh.abs() * (e * rh).abs().mean(-1, keepdim=True)) / size + d(dro).abs()), "dr")
    close(dw, (d(dn) * rh).sum(0), 100 * U * (d(dn) * rh).abs().sum(0), "dw_pre")
    y, ro = cuda(30, width, gen=gen, dtype=BF16), torch.empty_like(r)
    op = sequence.BlockNorm("bf16", width, residual="f32")
    op.forward(r, y, None, None, None, ro, None)
    v = d(y) / R.rms(d(y), 1e-6)
    close(ro, d(r) + v, 64 * U * (d(r).abs() + v.abs()), "r_out")


@pytest.mark.parametrize("width", [256, 333])
def test_norm_in_place(width):
    gen = torch.Generator("cuda").manual_seed(width)
    r, y = cuda(50, width, gen=gen, dtype=BF16), cuda(50, width, gen=gen, dtype=BF16)
    op = sequence.BlockNorm("bf16", width)
    ro, n, n2 = (torch.empty_like(r) for _ in range(3))
    op.forward(r, y, None, None, None, ro, n)
    dr, dy, dy2 = (torch.empty_like(r) for _ in range(3))
    dro, dn = cuda(50, width, gen=gen, dtype=BF16), cuda(50, width, gen=gen, dtype=BF16)
    op.backward(ro, y, None, None, None, dro, dn, dr, dy, None, None, None, None)
    op.forward(r, y, None, None, None, r, n2)
    op.backward(ro, y, None, None, None, dro, dn, dro, dy2, None, None, None, None)
    assert torch.equal(r, ro) and torch.equal(n, n2) and torch.equal(dro, dr) and torch.equal(dy, dy2)


def test_norm_of_no_rows():
    op = sequence.BlockNorm("f32", 64, gate="silu")
    e = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    op.forward(e, e, e, w, w, e.clone(), e.clone())
    dw, dv = torch.full((64,), 7.0, device="cuda"), torch.full((64,), 7.0, device="cuda")
    ws = torch.empty(op.workspace_bytes(0), dtype=torch.uint8, device="cuda")
    op.backward(e, e, e, w, w, None, e.clone(), e.clone(), e.clone(), e.clone(), dw, dv, ws)
    assert (dw == 0).all() and (dv == 0).all()


# ---- edges ---------------------------------------------------------------------------


def block(tokens, channels, n, dtype=BF16, complement=True, seed=0):
    """A recurrence's call of equal sequences: (op, inputs, buffers)."""
    gen = torch.Generator("cuda").manual_seed(seed)
    x, f, dh = cuda(tokens, channels, gen=gen, dtype=dtype), cuda(tokens, channels, gen=gen, dtype=dtype, scale=2.0), \
        cuda(tokens, channels, gen=gen, dtype=dtype)
    cu = torch.tensor([tokens * i // n for i in range(n + 1)], dtype=torch.int32, device="cuda")
    op = sequence.GatedRecurrence(dtype, channels, complement)
    ws = torch.empty(max(op.workspace_bytes(tokens, n), op.backward_workspace_bytes(tokens, n)), dtype=torch.uint8, device="cuda")
    return op, x, f, dh, 2 + cuda(channels, gen=gen), cu, ws


def both(op, x, f, dh, bias, cu, ws, keep=False, stream=None):
    """Outputs of a forward and a backward call."""
    tokens, channels, n = x.shape[0], x.shape[1], cu.numel() - 1
    h, dx, df = (torch.zeros_like(x) for _ in range(3))
    state, into, dbias = torch.zeros(n, channels, device="cuda"), torch.zeros(n, channels, device="cuda"), torch.zeros(channels, device="cuda")
    saved = torch.zeros(op.saved_rows(tokens, n), channels, device="cuda")
    kept = {"keep_" + k: sequence.Rows8.empty(tokens, channels) for k in "xf"} if keep else {}

    def run():
        op.forward(x, f, bias, cu, h, state_out=state, saved=saved, workspace=ws, stream=stream, **kept)
        op.backward(kept.get("keep_x", x), kept.get("keep_f", f), bias, cu, saved, dh, dx, df, dbias, dstate_in=into,
                    workspace=ws, stream=stream)

    return run, (h, state, dx, df, dbias, into)


@pytest.mark.parametrize("tokens,channels,n,keep", [(40000, 64, 1, False), (20000, 700, 1, True), (9000, 1024, 7, False),
                                                    (4000, 333, 3, False)])
def test_recurrence_repeats_to_the_bit(tokens, channels, n, keep):
    call = block(tokens, channels, n, seed=tokens)
    run, out = both(*call, keep=keep)
    run()
    first = [t.clone() for t in out]
    for _ in range(40):
        run()
    torch.cuda.synchronize()
    assert abi.lib.to_device_status(1) == 0
    for a, b in zip(first, out):
        assert torch.equal(a, b)


def test_recurrence_many_sequences_as_one_by_one():
    """Sequences taken side by side, of very different lengths, against each as a call of its own."""
    lengths = [5000, 1, 0, 130, 2000, 129, 128, 0, 700, 3, 1500, 64, 900]
    gen = torch.Generator("cuda").manual_seed(5)
    tokens, n = sum(lengths), len(lengths)
    op, x, f, dh, bias, _, _ = block(tokens, 200, 1, dtype=F32, seed=5)
    ends = [sum(lengths[:i]) for i in range(n + 1)]
    ws = torch.empty(max(op.workspace_bytes(tokens, n), op.backward_workspace_bytes(tokens, n)), dtype=torch.uint8, device="cuda")
    run, out = both(op, x, f, dh, bias, torch.tensor(ends, dtype=torch.int32, device="cuda"), ws)
    run()
    for i in range(n):
        a, b = ends[i], ends[i + 1]
        one = torch.tensor([0, b - a], dtype=torch.int32, device="cuda")
        single, want = both(op, x[a:b], f[a:b], dh[a:b], bias, one, ws)
        single()
        for got, w in zip((out[0][a:b], out[1][i:i + 1], out[2][a:b], out[3][a:b], out[5][i:i + 1]), (*want[:4], want[5])):
            assert torch.equal(got, w), i


def test_calls_on_two_streams_and_on_the_current_one():
    calls = [block(6000, 256, 2, seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    want = []
    for call in calls:
        run, out = both(*call)
        run()
        want.append([t.clone() for t in out])
    torch.cuda.synchronize()
    runs = [both(*call, stream=s.cuda_stream) for call, s in zip(calls, streams)]
    torch.cuda.synchronize()
    for _ in range(10):
        for run, _ in runs:
            run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    run, out = both(*calls[0][:-1], torch.empty_like(calls[0][-1]))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):  # no stream given: torch's current one
        run()
    torch.cuda.synchronize()
    for w, (_, got) in zip(want + want[:1], runs + [(None, out)]):
        for a, b in zip(w, got):
            assert torch.equal(a, b)


def test_captured_calls_replay():
    """Two graphs that share a workspace, and new inputs between replays."""
    call = block(3000, 256, 3)
    run, out = both(*call, keep=True)
    norm = sequence.BlockNorm("bf16", 256, gate="silu")
    gen = torch.Generator("cuda").manual_seed(9)
    r, g, ro, n = (cuda(3000, 256, gen=gen, dtype=BF16) for _ in range(4))
    dr, dy, dg = (torch.zeros_like(r) for _ in range(3))
    dw, dv = torch.zeros(256, device="cuda"), torch.zeros(256, device="cuda")
    ws = torch.empty(norm.workspace_bytes(3000), dtype=torch.uint8, device="cuda")

    def step():
        run()
        norm.forward(r, out[0], g, None, None, ro, n)
        norm.backward(ro, out[0], g, None, None, r, n, dr, dy, dg, dw, dv, ws)

    every = (*out, ro, n, dr, dy, dg, dw, dv)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
    for seed in (1, 2):
        call[1].copy_(cuda(3000, 256, gen=torch.Generator("cuda").manual_seed(seed), dtype=BF16))
        step()
        want = [t.clone() for t in every]
        for graph in graphs:
            for t in every:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, every):
                assert torch.equal(a, b)


def test_autograd_sees_what_is_written():
    op, x, f, dh, bias, cu, ws = block(64, 32, 1)
    h, state = torch.zeros_like(x), torch.zeros(1, 32, device="cuda")
    kept = sequence.Rows8.empty(64, 32)
    before = [t._version for t in (h, state, *kept)]
    op.forward(x, f, bias, cu, h, state_out=state, keep_x=kept)
    assert [t._version for t in (h, state, *kept)] == [v + 1 for v in before]


@pytest.mark.parametrize("at", [620, 621, 623, 626])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinities_stay_with_what_they_reach(dtype, at):
    """An infinite or NaN value reaches its channel's later tokens (gradients: the earlier ones) and no others."""
    op, x, f, dh, bias, cu, ws = block(1000, 96, 2, dtype=dtype, seed=4)
    run, out = both(op, x, f, dh, bias, cu, ws)
    run()
    want = [t.clone() for t in out]
    x[300, 7], f[at, 40], dh[200, 70] = float("inf"), float("nan"), float("nan")
    run()
    h, state, dx, df, dbias, into = out
    spoilt = torch.zeros(1000, 96, dtype=torch.bool, device="cuda")
    spoilt[300:500, 7] = spoilt[at:, 40] = True
    assert not torch.isfinite(h[spoilt]).any() and torch.equal(h[~spoilt], want[0][~spoilt])
    assert not torch.isfinite(state[0, 7]) and not torch.isfinite(state[1, 40])
    assert torch.isfinite(state[0, torch.arange(96) != 7]).all()
    back = torch.zeros_like(spoilt)
    back[:201, 70] = back[500:at + 1, 40] = True
    assert not torch.isfinite(dx[back]).any() and torch.equal(dx[~back], want[2][~back])
    assert not torch.isfinite(into[0, 70]) and not torch.isfinite(into[1, 40])
    clean = torch.ones(96, dtype=torch.bool, device="cuda")
    clean[[7, 40, 70]] = False
    assert torch.equal(df[:, clean], want[3][:, clean]) and torch.equal(dbias[clean], want[4][clean])


def test_gates_at_their_ends():
    """Tokens that forget everything or nothing are exact, and what is left of a far decayed state keeps its digits."""
    op = sequence.GatedRecurrence("f32", 4)
    x = torch.zeros(700, 4, device="cuda")
    f = torch.full((700, 4), 30.0, device="cuda")
    f[:, 1] = float("inf")
    f[350:, 2] = -13.0  # a = 2.3e-6 at every token: three leave 1e-17 of the state
    f[353:, 2] = 30.0
    f[400, 3], x[400, 3] = float("-inf"), 1e-3
    state = torch.tensor([[2.0, 3.0, 5.0, 1e4]], device="cuda")
    h, left = torch.empty_like(x), torch.empty_like(state)
    ws = torch.empty(op.workspace_bytes(700, 1), dtype=torch.uint8, device="cuda")
    op.forward(x, f, None, torch.tensor([0, 700], dtype=torch.int32, device="cuda"), h, state_in=state, state_out=left, workspace=ws)
    assert h[-1, 1] == 3.0 and left[0, 1] == 3.0
    want = 5.0 * torch.sigmoid(torch.tensor(-13.0, dtype=torch.float64)) ** 3
    for got in (h[-1, 2], left[0, 2]):  # (700 tokens that forget 1e-13 each)
        assert abs(float(got) / float(want) - 1) < (3 * (13 + 16) + 700 * 2) * U
    assert h[400, 3] == x[400, 3] and abs(float(left[0, 3]) / 1e-3 - 1) < 300 * 4 * U


@pytest.mark.parametrize("complement", [True, False])
def test_gradients_against_differences(complement):
    """dx, df, dbias and dstate against central differences of the 64-bit form, along random directions."""
    lengths = [150, 0, 40]
    op, x, f, dh, bias, _, ws = block(190, 24, 1, dtype=F32, complement=complement, seed=8)
    gen = torch.Generator("cuda").manual_seed(8)
    state, dstate = cuda(3, 24, gen=gen), cuda(3, 24, gen=gen)
    cu = torch.tensor([0, 150, 150, 190], dtype=torch.int32, device="cuda")
    h, dx, df = (torch.empty_like(x) for _ in range(3))
    saved, into, dbias = torch.empty(op.saved_rows(190, 3), 24, device="cuda"), torch.empty_like(state), torch.empty_like(bias)
    ws = torch.empty(max(op.workspace_bytes(190, 3), op.backward_workspace_bytes(190, 3)), dtype=torch.uint8, device="cuda")
    op.forward(x, f, bias, cu, h, state_in=state, saved=saved, workspace=ws)
    op.backward(x, f, bias, cu, saved, dh, dx, df, dbias, dstate_out=dstate, dstate_in=into, workspace=ws)
    at = [d(t) for t in (x, f, bias, state)]

    def loss(v):
        hh, _, left, *_ = R.recurrence(v[0], v[1], v[2], lengths, v[3], complement)
        return float((hh * d(dh)).sum() + (left * d(dstate)).sum())

    cpu = torch.Generator().manual_seed(8)
    for k, grad in enumerate((dx, df, dbias, into)):
        way = torch.randn(at[k].shape, generator=cpu, dtype=torch.float64)
        step = 1e-5
        ends = [loss([v + s * step * way if j == k else v for j, v in enumerate(at)]) for s in (1, -1)]
        # differences: step^2 of the third derivative, and the loss's rounding over the step; f32: its digits
        slope, got = (ends[0] - ends[1]) / (2 * step), float((d(grad) * way).sum())
        room = 1e-6 * float((d(grad) * way).abs().sum()) + 1e-6 * abs(slope) + 1e-6
        assert abs(slope - got) < 200 * room, (k, slope, got)


def test_norm_rows_keep_to_themselves():
    """An infinity or NaN in a row leaves the other rows as they are."""
    gen = torch.Generator("cuda").manual_seed(2)
    op = sequence.BlockNorm("bf16", 264, residual="f32", gate="sigmoid")
    r, y, g = cuda(20, 264, gen=gen), cuda(20, 264, gen=gen, dtype=BF16), cuda(20, 264, gen=gen, dtype=BF16)
    out = []
    for _ in range(2):
        ro, n = torch.empty_like(r), torch.empty_like(y)
        op.forward(r, y, g, None, None, ro, n)
        out.append((ro, n))
        y[3, 5], g[7, 100], r[11, 0] = float("inf"), float("nan"), float("-inf")
    rows = torch.ones(20, dtype=torch.bool, device="cuda")
    rows[[3, 7, 11]] = False
    for a, b in zip(*out):
        assert torch.equal(a[rows], b[rows]) and not torch.isfinite(b[~rows]).all(1).any()


def test_largest_gates_and_smallest_rows():
    """Gates of +-100, rows of zeros without eps (n has no value there) and with it."""
    g = torch.tensor([[100.0, -100.0, 0.0, 30.0]], device="cuda")
    y = torch.ones(1, 4, device="cuda")
    for gate in ("sigmoid", "silu"):
        op = sequence.BlockNorm("f32", 4, gate=gate, post_norm=False)
        r, ro, n = torch.zeros(1, 4, device="cuda"), torch.empty(1, 4, device="cuda"), torch.empty(1, 4, device="cuda")
        op.forward(r, y, g, None, None, ro, n)
        p = torch.sigmoid(d(g))
        want = p if gate == "sigmoid" else d(g) * p
        # (where sigmoid(g) lies below 2^-126 the kernel has 2^-126)
        close(ro, want, (2 * d(g).abs() + 16) * U * want.abs() + 2.0 ** -126 * d(g).abs().clamp(min=1), gate)
    op = sequence.BlockNorm("f32", 4)
    zero = torch.zeros(2, 4, device="cuda")
    op.forward(zero, zero, None, None, None, ro2 := torch.empty(2, 4, device="cuda"), n2 := torch.empty(2, 4, device="cuda"))
    assert (ro2 == 0).all() and (n2 == 0).all()
