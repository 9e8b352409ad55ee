"""Waits of the gated recurrence that run out: the launch ends, the status says so, nothing wrong passes for a result,
and the next call is right."""
import pytest

torch = pytest.importorskip("torch")
from tensoroperations_b200 import abi, sequence  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def limits():
    """Sets the limits, and takes them back."""
    yield lambda maps, tiles: abi.check(abi.lib.to_gated_recurrence_wait_limits(maps, tiles), "limits")
    torch.cuda.synchronize()
    abi.lib.to_gated_recurrence_wait_limits(-1, -1)
    abi.lib.to_device_status(1)


def calls(dtype, channels, lengths, keep):
    gen = torch.Generator("cuda").manual_seed(channels)
    tokens, n = sum(lengths), len(lengths)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, f, dh = (normal(tokens, channels).to(dtype) for _ in range(3))
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    op = sequence.GatedRecurrence(dtype, channels)
    ws = torch.empty(max(op.workspace_bytes(tokens, n), op.backward_workspace_bytes(tokens, n)), dtype=torch.uint8, device="cuda")
    kept = {k: sequence.Rows8.empty(tokens, channels) for k in ("keep_x", "keep_f")} if keep else {}

    def forward():
        h, left = torch.full_like(x, torch.nan), torch.full((n, channels), torch.nan, device="cuda")
        saved = torch.full((op.saved_rows(tokens, n), channels), torch.nan, device="cuda")
        op.forward(x, f, None, cu, h, state_out=left, saved=saved, workspace=ws, **kept)
        torch.cuda.synchronize()
        return h, left, saved

    def backward(saved):
        dx, df = torch.full_like(x, torch.nan), torch.full_like(x, torch.nan)
        into, dbias = torch.full((n, channels), torch.nan, device="cuda"), torch.full((channels,), torch.nan, device="cuda")
        op.backward(kept.get("keep_x", x), kept.get("keep_f", f), None, cu, saved, dh, dx, df, dbias, dstate_in=into, workspace=ws)
        torch.cuda.synchronize()
        return dx, df, into, dbias

    return forward, backward


@pytest.mark.parametrize("dtype,channels,lengths,keep", [
    (BF16, 64, [20000], False),  # few chains: tickets as late as can be
    (BF16, 2048, [3000, 0, 1, 2500, 4000], True),
    (F32, 96, [9000, 700], False),
    (F32, 333, [5000, 130, 3000], True),  # rows and codes that TMA does not take
    (BF16, 4096, [1500] * 4, False),
    (F32, 128, [128, 0, 100, 128, 3], True)])  # no maps to wait for
@pytest.mark.parametrize("which", ["maps", "tiles"])
def test_waits_that_run_out(limits, which, dtype, channels, lengths, keep):
    if which == "maps" and max(lengths) <= 128:
        pytest.skip("no sequence waits for maps")
    forward, backward = calls(dtype, channels, lengths, keep)
    want = forward()
    want_back = backward(want[2])
    assert abi.lib.to_device_status(1) == 0
    for call, right in ((forward, want), (lambda: backward(want[2]), want_back)):
        limits(*((0, -1) if which == "maps" else (-1, 0)))
        got = call()
        assert abi.lib.to_device_status(1) == abi.TO_ERR_TIMEOUT
        assert abi.lib.to_device_status(1) == 0
        spoilt = 0
        for a, b in zip(got, right):  # (memory of NaN before the call: what has not come is NaN)
            fine = ~torch.isnan(a)
            assert torch.equal(a[fine], b[fine])
            spoilt += int((~fine & ~torch.isnan(b)).sum())
        assert spoilt > 0
        limits(-1, -1)
        for a, b in zip(call(), right):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        assert abi.lib.to_device_status(1) == 0


def test_what_needs_no_maps_is_not_touched_by_their_limit(limits):
    """Sequences of one segment wait for none."""
    forward, backward = calls(F32, 200, [128, 1, 0, 77, 128], False)
    want = forward()
    limits(0, -1)
    got = forward()
    assert abi.lib.to_device_status(1) == 0
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
