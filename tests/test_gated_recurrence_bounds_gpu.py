"""The gated recurrence within bounds that follow its errors token by token (gated_recurrence_bounds), on gates like a
trained layer's and on wide ones: whole segments, long chains, rows in 8 bits."""
import pytest

torch = pytest.importorskip("torch")
from tensoroperations_b200 import abi, sequence  # noqa: E402
from tests import gated_recurrence_bounds as B, recurrent_block_oracle as R  # noqa: E402
from tests.recurrent_block_oracle import U, d  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def within(got, want, tol, dtype, what):
    """Within tol and one rounding of what it then is."""
    got, want = d(got), d(want)
    room = tol + (R.half(dtype) * (want.abs() + tol) if dtype != F32 else 0)
    share = (got - want).abs() / room.clamp(min=1e-300)
    assert torch.isfinite(got).all() and (share <= 1).all(), f"{what}: {share.max():.2f} of the bound"


def check(dtype, channels, lengths, gates, complement=True, keep=False, states=True, packed=False):
    gen = torch.Generator("cuda").manual_seed(channels + sum(lengths))
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    tokens, n = sum(lengths), len(lengths)
    rows = normal(tokens, 2 * channels + (3 if packed else 0)).to(dtype)
    x, f = rows[:, -2 * channels:-channels], rows[:, -channels:]
    bias = 1 + 7 * torch.rand(channels, generator=gen, device="cuda") if gates == "layer" else None
    if gates == "wide":
        f *= 4
    state = normal(n, channels) if states else None
    dstate = normal(n, channels) if states else None
    dh = normal(tokens, channels).to(dtype)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    op = sequence.GatedRecurrence(dtype, channels, complement)
    h, dx, df = (torch.empty(tokens, channels, dtype=dtype, device="cuda") for _ in range(3))
    left, into = (torch.empty(n, channels, device="cuda") for _ in range(2)) if states else (None, None)
    saved, dbias = torch.empty(op.saved_rows(tokens, n), channels, device="cuda"), torch.empty(channels, device="cuda")
    ws = torch.empty(op.workspace_bytes(tokens, n), dtype=torch.uint8, device="cuda") if op.workspace_bytes(tokens, n) else None
    kept = {k: sequence.Rows8.empty(tokens, channels) for k in ("keep_x", "keep_f")} if keep else {}
    op.forward(x, f, bias, cu, h, state_in=state, state_out=left, saved=saved, workspace=ws, **kept)
    ws = torch.empty(op.backward_workspace_bytes(tokens, n), dtype=torch.uint8, device="cuda")
    op.backward(kept.get("keep_x", x), kept.get("keep_f", f), bias, cu, saved, dh, dx, df, dbias, dstate_out=dstate, dstate_in=into,
                workspace=ws)
    assert abi.lib.to_device_status(1) == 0

    zero = torch.zeros(n, channels, dtype=torch.float64)
    s0, ds0, x0, f0, dh0 = zero if state is None else d(state), zero if dstate is None else d(dstate), d(x), d(f), d(dh)
    b0 = 0 if bias is None else d(bias)
    want, before, wleft, a, z = R.recurrence(x0, f0, None if bias is None else b0, lengths, s0, complement)
    after, ahead = B.values(x0, f0 + b0, a, z, want, before, lengths, s0, complement)
    within(h, want, after, dtype, "h")
    if states:
        last, at = zero.clone(), 0
        for k, m in enumerate(lengths):
            at += m
            if m:
                last[k] = after[at - 1] + 10 * U * wleft[k].abs()  # (joined from the chains' maps)
        within(left, wleft, last, F32, "state")
    if keep:  # gradients of the values kept, from the states that the forward pass had every 128 tokens
        x0, f0 = (R.unpack8(*R.pack8(t)) for t in (x, f))
        pieces = [min(B.SEGMENT, m - i) for m in lengths for i in range(0, m, B.SEGMENT)]
        heads = torch.tensor([0] + pieces).cumsum(0)[:-1]
        enter, room = before[heads], ahead[heads]
        hh, before, _, a, z = R.recurrence(x0, f0, None if bias is None else b0, pieces, enter, complement)
        _, ahead = B.values(x0, f0 + b0, a, z, hh, before, pieces, enter, complement, heads=room)
    wx, wf, wb, winto, G = R.recurrence_grad(x0, a, z, before, lengths, dh0, ds0, complement)
    g0 = f0 + b0
    of_g, of_into = B.gradients(g0, a, z, G, dh0, ds0, lengths)
    off, part = B.gate(g0) + 2 * U, (before - x0 if complement else before)
    within(dx, wx, z * of_g + off * wx.abs() if complement else of_g, dtype, "dx")
    size = before.abs() + (x0.abs() if complement else 0)
    of_f = a * z * (of_g * part.abs() + (G.abs() + of_g) * (ahead + 2 * U * size)) + (2 * off + 3 * U) * wf.abs()
    within(df, wf, of_f, dtype, "df")
    # sums: 16 tokens, 8 chains, then in 64 bits
    within(dbias, wb, of_f.sum(0) + 26 * U * wf.abs().sum(0), F32, "dbias")
    if states:
        within(into, winto, of_into + 10 * U * winto.abs(), F32, "dstate_in")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gates", ["layer", "unit", "wide"])
@pytest.mark.parametrize("keep", [False, True])
def test_whole_segments(dtype, gates, keep):
    check(dtype, 128, [640, 128, 0, 129, 1, 256], gates, keep=keep)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gates", ["layer", "unit"])
def test_long_chains(dtype, gates):
    check(dtype, 64, [5000, 77, 2100], gates)


@pytest.mark.parametrize("gates", ["layer", "wide"])
def test_plain_input(gates):
    check(F32, 72, [700, 5, 300], gates, complement=False)


@pytest.mark.parametrize("channels", [33, 65, 100])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_odd_rows(channels, dtype):
    check(dtype, channels, [200, 0, 131, 40], "layer", keep=channels == 65, packed=True)


@pytest.mark.parametrize("lengths", [[128], [64, 64], [100, 0, 28], [127, 1], [1] * 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_segment_in_all_without_states(lengths, dtype):
    """Calls of 128 tokens at most need no workspace forwards."""
    assert sequence.GatedRecurrence(dtype, 50).workspace_bytes(sum(lengths), len(lengths)) == 0
    check(dtype, 50, lengths, "unit", states=False)
