"""How exact the gated recurrence's gates are, value by value."""
import pytest

torch = pytest.importorskip("torch")
from tensoroperations_b200 import abi, sequence  # noqa: E402
from tests.recurrent_block_oracle import U, d  # noqa: E402

pytestmark = pytest.mark.gpu

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
