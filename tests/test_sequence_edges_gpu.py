"""The sequence operators at the edges of their ranges, against definitions in float64:
heads split over warps.

Tolerances are those of test_sequence_gpu (derived there from the types alone) unless a
test says otherwise.
"""
import pytest

from test_sequence_gpu import TOL, close, qk_definition, qk_inputs

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
