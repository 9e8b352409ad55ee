"""How exact the gated recurrence's gates are, value by value, and that they go by their own channel alone."""
import pytest

torch = pytest.importorskip("torch")
from tensoroperations_b200 import abi, sequence  # noqa: E402
from tests.recurrent_block_oracle import U, d, half  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def whole(op, x, f, bias, dh, state=None, cu=None):
    """h, dx, df, dbias, dstate_in of one call on whole segments."""
    tokens, channels = x.shape
    cu = torch.tensor([0, tokens] if cu is None else cu, dtype=torch.int32, device="cuda")
    n = cu.numel() - 1
    ws = torch.empty(max(op.workspace_bytes(tokens, n), op.backward_workspace_bytes(tokens, n)), dtype=torch.uint8, device="cuda")
    h, dx, df = (torch.empty_like(x) for _ in range(3))
    saved, dbias = torch.empty(op.saved_rows(tokens, n), channels, device="cuda"), torch.empty(channels, device="cuda")
    into = torch.empty(n, channels, device="cuda")
    op.forward(x, f, bias, cu, h, state_in=state, saved=saved, workspace=ws)
    op.backward(x, f, bias, cu, saved, dh, dx, df, dbias, dstate_in=into, workspace=ws)
    assert abi.lib.to_device_status(1) == 0
    return h, dx, df, dbias, into


def gate_room(g):
    """Of the smaller of a and 1 - a, and of their product, relative.  The argument's sum and product: |g| U each, log2 e
    |g| U; 2^t: 2^-22 (4 U); the sum 1 + 2^t U, its reciprocal 2^-23 (2 U), the product U."""
    return (3 * g.abs() + 8) * U


@pytest.mark.parametrize("low,high", [(-2.77, -2.5), (-2.5, -1.5), (-1.5, 1.5), (1.5, 2.77), (-12.0, -2.77), (2.77, 12.0)])
def test_gates_keep_their_digits(low, high):
    """One token a segment has the gate to be seen, the others keep everything (1 - a = 1.4e-11): with x = 0 and a state
    of 1, h after it is a, and with dh = 1 at it alone dx = 1 - a and df = a (1 - a)."""
    channels, tokens, at = 2048, 384, 200
    g = torch.linspace(low, high, channels, dtype=torch.float64).float()
    f = torch.full((tokens, channels), 25.0, device="cuda")
    f[at] = g.cuda()
    x, dh = torch.zeros_like(f), torch.zeros_like(f)
    dh[at] = 1
    op = sequence.GatedRecurrence("f32", channels)
    h, dx, df, dbias, into = whole(op, x, f, None, dh, state=torch.ones(1, channels, device="cuda"))
    g = g.double()
    a, z = torch.sigmoid(g), torch.sigmoid(-g)
    # the larger of the two is 1 - the smaller one: a rounding, and the smaller one's error, which is no larger relative to it
    room = gate_room(g) + 2 * U
    # 383 tokens that keep 1 - 1.4e-11, each of which may round (joined maps: 3 products of segments)
    rest = 384 * 1.4e-11 + 8 * U
    for name, got, want, tol in (("a", h[at], a, room + rest), ("1 - a", dx[at], z, room), ("a (1 - a)", df[at], a * z, 2 * room + rest),
                                 ("a behind the segment", h[-1], a, room + rest), ("state's gradient", into[0], a, room + rest)):
        off = (d(got) / want - 1).abs()
        k = int((off / tol).argmax())
        assert (off <= tol).all(), f"{name} of {g[k]:.6f}: off by {off[k] / U:.1f} U of {tol[k] / U:.1f} U, rms {off.square().mean().sqrt() / U:.2f} U"


@pytest.mark.parametrize("bias", [20.0, 60.0, -200.0])
def test_gates_where_bias_and_gate_cancel(bias):
    """The argument is f + bias, whose rounding is relative to the sum: prompts and single tokens compute the same gate."""
    channels = 1024
    off = torch.linspace(-1.0, 1.0, channels, device="cuda")
    b = torch.full((channels,), bias, device="cuda")
    f = torch.empty(256, channels, device="cuda")
    f[:] = 25.0 - bias
    f[130] = off - bias
    g = d(f)[130] + d(b)
    x, dh = torch.zeros_like(f), torch.zeros_like(f)
    dh[130] = 1
    op = sequence.GatedRecurrence("f32", channels)
    h, dx, df, _, _ = whole(op, x, f, b, dh, state=torch.ones(1, channels, device="cuda"))
    a, z = torch.sigmoid(g), torch.sigmoid(-g)
    room = gate_room(g) + 2 * U
    rest = 256 * 1.4e-11 + 8 * U
    state, out = torch.ones(1, channels, device="cuda"), torch.empty(1, channels, device="cuda")
    op.step(x[:1], f[130:131], b, state, out)
    for name, got, want, tol in (("step", out[0], a, room), ("a", h[130], a, room + rest), ("1 - a", dx[130], z, room),
                                 ("a (1 - a)", df[130], a * z, 2 * room + rest)):
        rel = (d(got) / want - 1).abs()
        assert (rel <= tol).all(), f"{name}: off by {(rel / U).max():.1f} U, {(rel / tol).max():.2f} of the bound"


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("keep", [False, True])
def test_a_channel_goes_by_its_own_gates(dtype, keep):
    """Gates that forget (or are NaN) in one channel leave every bit of the others, on gates like a trained layer's."""
    tokens, channels = 640, 192
    gen = torch.Generator("cuda").manual_seed(3)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    x, f, dh = normal(tokens, channels), normal(tokens, channels), normal(tokens, channels)
    bias = 3.5 + 4 * torch.rand(channels, generator=gen, device="cuda")
    assert ((f.float() + bias) > -2.0).all()
    op = sequence.GatedRecurrence(dtype, channels)

    def call():
        if not keep:
            return whole(op, x, f, bias, dh, cu=[0, 384, 640])
        cu = torch.tensor([0, 384, 640], dtype=torch.int32, device="cuda")
        ws = torch.empty(max(op.workspace_bytes(tokens, 2), op.backward_workspace_bytes(tokens, 2)), dtype=torch.uint8, device="cuda")
        h, dx, df = (torch.empty_like(x) for _ in range(3))
        saved, dbias = torch.empty(op.saved_rows(tokens, 2), channels, device="cuda"), torch.empty(channels, device="cuda")
        kx, kf = sequence.Rows8.empty(tokens, channels), sequence.Rows8.empty(tokens, channels)
        op.forward(x, f, bias, cu, h, saved=saved, keep_x=kx, keep_f=kf, workspace=ws)
        into = torch.empty(2, channels, device="cuda")
        op.backward(kx, kf, bias, cu, saved, dh, dx, df, dbias, dstate_in=into, workspace=ws)
        return h, dx, df, dbias, into

    first = call()
    changed = [5, 64, 130]
    f[:, 5] = -8.0  # forgets at every token
    f[100, 64], f[450, 64] = -12.0, -9.0  # at two of them
    f[300, 130] = float("nan")
    # (in 8 bits a group of 32 shares its scale, and a NaN its whole group)
    spoilt = [c for c in range(channels) if (c // 32 if keep else c) in {(k // 32 if keep else k) for k in changed}]
    clean = torch.ones(channels, dtype=torch.bool, device="cuda")
    clean[spoilt] = False
    for a, b in zip(first, call()):
        assert torch.equal(a[..., clean], b[..., clean])


@pytest.mark.parametrize("at", [128, 200, 201, 203, 255, 383])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_nan_gate_spoils_no_earlier_token(dtype, at):
    """In a whole segment of gates that keep: tokens before it (gradients: behind it) keep every bit."""
    tokens, channels = 512, 64
    gen = torch.Generator("cuda").manual_seed(at)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    x, f, dh = normal(tokens, channels), normal(tokens, channels), normal(tokens, channels)
    bias = torch.full((channels,), 5.0, device="cuda")
    op = sequence.GatedRecurrence(dtype, channels)
    h, dx, df, _, _ = whole(op, x, f, bias, dh)
    f[at, 17] = float("nan")
    h2, dx2, df2, dbias, into = whole(op, x, f, bias, dh)
    kept = torch.ones(tokens, channels, dtype=torch.bool, device="cuda")
    kept[at:, 17] = False
    assert torch.equal(h[kept], h2[kept]) and not torch.isfinite(h2[~kept]).any()
    kept[:] = True
    kept[:at + 1, 17] = False
    assert torch.equal(dx[kept], dx2[kept]) and not torch.isfinite(dx2[~kept]).any()
    kept[:, 17] = False  # (df needs the state before a token too)
    assert torch.equal(df[kept], df2[kept]) and not torch.isfinite(into[0, 17]) and not torch.isfinite(dbias[17])


def test_bf16_gates_round_once():
    """bf16 rows: states in f32 have the gates' digits, h takes its one rounding."""
    channels, tokens = 512, 256
    f = torch.full((tokens, channels), 25.0, device="cuda", dtype=BF16)
    f[140] = torch.linspace(-2.76, -1.0, channels).to(BF16).cuda()
    op = sequence.GatedRecurrence("bf16", channels)
    h, left = torch.empty_like(f), torch.empty(1, channels, device="cuda")
    ws = torch.empty(op.workspace_bytes(tokens, 1), dtype=torch.uint8, device="cuda")
    op.forward(torch.zeros_like(f), f, None, torch.tensor([0, tokens], dtype=torch.int32, device="cuda"), h,
               state_in=torch.ones(1, channels, device="cuda"), state_out=left, workspace=ws)
    g = d(f)[140]
    a = torch.sigmoid(g)
    tol = gate_room(g) + 2 * U + 256 * 1.4e-11 + 8 * U
    off = (d(left)[0] / a - 1).abs()
    assert (off <= tol).all(), f"state: off by {(off / U).max():.1f} U, {(off / tol).max():.2f} of the bound"
    assert ((d(h)[140] / a - 1).abs() <= tol + half(BF16)).all()
