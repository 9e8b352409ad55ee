"""What the recurrent block's operators refuse, without a GPU: descriptors, sizes, strides, alignments and
shared memory are checked before anything is launched."""
import math

import pytest

from tensoroperations_b200 import abi

torch = pytest.importorskip("torch")
from tensoroperations_b200 import sequence  # noqa: E402

BOGUS = 0x100000  # an aligned address that nothing reads
FAR = [BOGUS + (n << 24) for n in range(12)]  # rows that lie apart
BAD, NO, ODD = abi.TO_ERR_INVALID_ARGUMENT, abi.TO_ERR_UNSUPPORTED, abi.TO_ERR_ALIGNMENT


@pytest.mark.parametrize("bad,status", [(dict(channels=0), NO), (dict(channels=65537), NO), (dict(channels=-3), NO)])
def test_recurrence_descriptors(bad, status):
    with pytest.raises(abi.ToError) as e:
        sequence.GatedRecurrence("bf16", **bad)
    assert e.value.status == status


@pytest.mark.parametrize("bad,status", [
    (dict(width=0), NO), (dict(width=16385), NO), (dict(scale=math.nan), BAD), (dict(scale=math.inf), BAD),
    (dict(eps=-1.0), BAD), (dict(eps=math.nan), BAD), (dict(dtype="f32", residual="bf16"), NO)])
def test_norm_descriptors(bad, status):
    with pytest.raises(abi.ToError) as e:
        sequence.BlockNorm(**{**dict(dtype="bf16", width=64), **bad})
    assert e.value.status == status


def test_python_refusals():
    for make in (lambda: sequence.GatedRecurrence("f16", 8), lambda: sequence.BlockNorm("f64", 8),
                 lambda: sequence.BlockNorm("bf16", 8, gate="relu"), lambda: sequence.Checkpoint8("int8", 8),
                 lambda: sequence.BlockNorm("bf16", 2 ** 40), lambda: sequence.GatedRecurrence("bf16", 2 ** 31)):
        with pytest.raises(ValueError):
            make()
    with pytest.raises(abi.ToError):
        sequence.Checkpoint8("bf16", 0)
    x, f32 = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, 64)
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        sequence.GatedRecurrence("bf16", 64).forward(x, x, None, cu, x)
    with pytest.raises(ValueError, match="CUDA"):
        sequence.GatedRecurrence("bf16", 64).step(x, x, None, f32, x)
    with pytest.raises(ValueError, match="CUDA"):
        sequence.BlockNorm("bf16", 64).forward(x, x, None, None, None, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        sequence.Checkpoint8("bf16", 64).pack(x, sequence.Rows8.empty(3, 64, "cpu"))
    kept = sequence.Rows8.empty(5, 65, "cpu")
    assert kept.codes.shape == (5, 65) and kept.scales.shape == (5, 3)


def rec_args(x=None, f=None, h=None, kx=(0, 0, 0, 0), kf=(0, 0, 0, 0), bias=0, cu=BOGUS, slots=0, s_in=0, s_out=0, saved=0,
             ws=0, n=0):
    r = [(FAR[k], 64, 0) if t is None else t for k, t in enumerate((x, f, h))]
    return sequence._REC_ARGS.pack(*r[0], *r[1], *r[2], *kx, *kf, bias, cu, slots, s_in, s_out, saved, ws, n)


@pytest.mark.parametrize("kw,want", [
    (dict(x=(0, 64, 0)), BAD), (dict(f=(FAR[1] + 1, 64, 0)), ODD), (dict(h=(FAR[2], 63, 0)), BAD),
    (dict(x=(FAR[0], -64, 0)), BAD), (dict(cu=0), BAD), (dict(cu=BOGUS + 2), ODD), (dict(bias=BOGUS + 1), ODD),
    (dict(slots=BOGUS + 3), ODD), (dict(s_in=BOGUS + 4), ODD), (dict(s_out=BOGUS + 8), ODD), (dict(saved=BOGUS + 4), ODD),
    (dict(kx=(FAR[5], 0, 64, 2)), BAD), (dict(kf=(FAR[5], FAR[6], 63, 2)), BAD), (dict(kf=(FAR[5], FAR[6], 64, 1)), BAD),
    (dict(h=(FAR[0], 64, 0)), BAD), (dict(h=(FAR[1] + 64 * 59 * 2, 64, 0)), BAD),  # rows that h shares with x, with f
    (dict(kx=(FAR[2], FAR[6], 64, 2)), BAD), (dict(kx=(FAR[5], FAR[0], 64, 2)), BAD),
    (dict(s_in=FAR[7], s_out=FAR[7] + 64), BAD), (dict(s_in=FAR[7], saved=FAR[7]), BAD),
])
def test_recurrence_refuses_before_any_launch(kw, want):
    op = sequence.GatedRecurrence("bf16", 64)
    assert abi.lib.to_gated_recurrence(op._desc(60, 1, 1), rec_args(**kw), 0) == want
    assert abi.lib.to_last_error()


def test_recurrence_other_refusals():
    op = sequence.GatedRecurrence("bf16", 64)
    run = abi.lib.to_gated_recurrence
    assert run(None, rec_args(), 0) == BAD and run(op._desc(60, 1), None, 0) == BAD
    assert run(op._desc(-1, 1), rec_args(), 0) == BAD and run(op._desc(60, -1), rec_args(), 0) == BAD
    assert run(op._desc(60, 70000), rec_args(), 0) == BAD and run(op._desc(2 ** 31, 1), rec_args(), 0) == BAD
    assert run(op._desc(60, 1, -1), rec_args(), 0) == BAD
    assert run(sequence._REC_DESC.pack(7, 64, 1, 1, 60, 1), rec_args(), 0) == NO
    assert run(sequence._REC_DESC.pack(2, 64, 1, 2, 60, 1), rec_args(), 0) == BAD
    # sequences that may be longer than a segment need a workspace
    assert op.workspace_bytes(100000, 1) > 0
    assert run(op._desc(100000, 1, 1), rec_args(), 0) == BAD and b"workspace" in abi.lib.to_last_error()
    need = op.workspace_bytes(100000, 1)
    assert run(op._desc(100000, 1, 1), rec_args(ws=FAR[11] + 64, n=need), 0) == ODD
    assert run(op._desc(100000, 1, 1), rec_args(ws=FAR[11], n=need - 1), 0) == BAD
    # nothing to do is not an error, whatever the pointers are
    assert run(op._desc(0, 0), rec_args(x=(0, 0, 0), f=(0, 0, 0), h=(0, 0, 0), cu=0), 0) == abi.TO_OK
    step = abi.lib.to_gated_recurrence_step
    assert step(op._desc(3, 0, 3), rec_args(), 0) == BAD  # no state
    assert step(op._desc(3, 0, 3), rec_args(s_out=BOGUS + 4), 0) == ODD
    assert step(op._desc(3, 0, 3), rec_args(s_out=FAR[8], h=(FAR[0], 64, 0)), 0) == BAD
    assert step(op._desc(0, 0), rec_args(x=(0, 0, 0)), 0) == abi.TO_OK

    def grad(x=FAR[0], x8=(0, 0, 0, 0), dx=FAR[3], df=FAR[4], saved=FAR[5], d_out=0, d_in=0, db=0, ws=0, n=0):
        rows = [(p, 64, 0) for p in (x, FAR[1], FAR[2], dx, df)]
        return sequence._REC_GRAD_ARGS.pack(*sum(rows, ()), *x8, 0, 0, 0, 0, 0, BOGUS, saved, d_out, d_in, db, ws, n)

    back = abi.lib.to_gated_recurrence_backward
    need = op.backward_workspace_bytes(60, 1)
    for kw, want in ((dict(saved=0), BAD), (dict(saved=BOGUS + 8), ODD), (dict(dx=FAR[0]), BAD), (dict(df=FAR[3]), BAD),
                     (dict(d_out=FAR[6], d_in=FAR[6]), BAD), (dict(d_in=FAR[5]), BAD), (dict(d_in=BOGUS + 4), ODD),
                     (dict(d_in=FAR[6], db=FAR[6] + 128), BAD), (dict(db=FAR[5]), BAD), (dict(db=BOGUS + 1), ODD),
                     (dict(x8=(FAR[7], 0, 64, 2)), BAD), (dict(x8=(FAR[3], FAR[7], 64, 2)), BAD)):
        assert back(op._desc(60, 1, 1), grad(ws=FAR[11], n=need, **kw), 0) == want, kw
    assert back(op._desc(60, 1, 1), grad(), 0) == BAD and b"workspace" in abi.lib.to_last_error()


def test_sizes_of_recurrence_buffers():
    op = sequence.GatedRecurrence("f32", 100)
    assert op.workspace_bytes(0, 0) == 0 and op.workspace_bytes(1, 1) == 0 and op.workspace_bytes(128, 9) == 0
    assert op.workspace_bytes(1 << 20, 1) % 256 == 0 and op.backward_workspace_bytes(1, 1) >= 400
    for tokens, n in ((0, 1), (1, 1), (128, 1), (129, 1), (5000, 7)):  # every segment of any lengths has a row
        assert op.saved_rows(tokens, n) >= n + (tokens - n) // 128
    assert abi.lib.to_gated_recurrence_workspace_bytes(None) == 0 and abi.lib.to_gated_recurrence_saved_rows(None) == 0
    assert abi.lib.to_gated_recurrence_backward_workspace_bytes(None) == 0
    assert abi.lib.to_block_norm_workspace_bytes(None, 5) == 0


def norm_args(r=FAR[0], y=FAR[1], g=FAR[2], ro=FAR[3], n=FAR[4], kr=(0, 0, 0, 0), ky=(0, 0, 0, 0), kg=(0, 0, 0, 0), w=0,
              stride=64):
    rows = [(p, stride, 0) if p else (0, 0, 0) for p in (r, y, g, ro, n)]
    return sequence._NORM_ARGS.pack(*sum(rows, ()), *kr, *ky, *kg, w, 0)


@pytest.mark.parametrize("kw,want", [
    (dict(r=0), BAD), (dict(g=0), BAD), (dict(ro=0), BAD), (dict(y=0), BAD), (dict(y=0, ro=0, g=0, n=0), BAD),
    (dict(n=FAR[4] + 1), ODD), (dict(w=BOGUS + 2), ODD), (dict(stride=63), BAD), (dict(n=FAR[1]), BAD), (dict(n=FAR[3]), BAD),
    (dict(ro=FAR[1]), BAD), (dict(ro=FAR[0] + 128), BAD), (dict(kr=(FAR[5], 0, 64, 2)), BAD),
    (dict(ky=(FAR[4], FAR[5], 64, 2)), BAD), (dict(kg=(FAR[5], FAR[2], 64, 2)), BAD)])
def test_norm_refuses_before_any_launch(kw, want):
    op = sequence.BlockNorm("bf16", 64, gate="silu")
    assert abi.lib.to_block_norm(op._desc, 9, norm_args(**kw), 0) == want
    assert abi.lib.to_last_error()


def test_norm_other_refusals():
    op, plain = sequence.BlockNorm("bf16", 64, gate="silu"), sequence.BlockNorm("bf16", 64)
    assert abi.lib.to_block_norm(None, 1, norm_args(), 0) == BAD and abi.lib.to_block_norm(op._desc, 1, None, 0) == BAD
    assert abi.lib.to_block_norm(op._desc, -1, norm_args(), 0) == BAD
    assert abi.lib.to_block_norm(plain._desc, 3, norm_args(), 0) == BAD  # a gate's rows without a gate
    assert abi.lib.to_block_norm(op._desc, 0, norm_args(r=0, y=0), 0) == abi.TO_OK
    for value in (4, -1):
        assert abi.lib.to_block_norm(sequence._NORM_DESC.pack(2, 2, 64, value, 1, 0, 1.0, 0.0), 0, norm_args(), 0) == BAD
    assert abi.lib.to_block_norm(sequence._NORM_DESC.pack(2, 2, 64, 0, 2, 0, 1.0, 0.0), 0, norm_args(), 0) == BAD
    # r_out, y, g, dr_out, dn, dr, dy, dg; then r8, y8, g8; w_post, w_pre, dw_post, dw_pre, workspace
    def grad(p, k=(0,) * 12, tail=(0, 0, 0, 0, 0, 0)):
        return sequence._NORM_GRAD_ARGS.pack(*sum([(x, 64, 0) if x else (0, 0, 0) for x in p], ()), *k, *tail)

    back, good = abi.lib.to_block_norm_backward, FAR[:8]
    for change, want in (({0: 0}, BAD), ({2: 0}, BAD), ({5: 0}, BAD), ({6: 0}, BAD), ({7: 0}, BAD), ({6: FAR[4]}, BAD),
                         ({7: FAR[6]}, BAD), ({5: FAR[0]}, BAD), ({6: FAR[6] + 1}, ODD)):
        p = [change.get(i, x) for i, x in enumerate(good)]
        assert back(op._desc, 9, grad(p), 0) == want, change
    assert back(op._desc, 9, grad(good, tail=(0, 0, FAR[8], 0, 0, 0)), 0) == BAD and b"workspace" in abi.lib.to_last_error()
    assert back(op._desc, 9, grad(good, tail=(0, 0, FAR[8] + 2, 0, FAR[9], 1 << 30)), 0) == ODD
    assert back(op._desc, 9, grad(good, tail=(0, 0, FAR[8], 0, FAR[9] + 8, 1 << 30)), 0) == ODD
    assert back(op._desc, 9, grad(good, tail=(0, 0, FAR[8], FAR[8] + 128, FAR[9], 1 << 30)), 0) == BAD  # weights' gradients that meet
    assert back(op._desc, 9, None, 0) == BAD and back(None, 9, grad(good), 0) == BAD


@pytest.mark.parametrize("x,p,want", [
    ((0, 64, 0), None, BAD), ((FAR[0] + 1, 64, 0), None, ODD), ((FAR[0], 63, 0), None, BAD), (None, (0, FAR[2], 64, 2), BAD),
    (None, (FAR[1], 0, 64, 2), BAD), (None, (FAR[1], FAR[2], 60, 2), BAD), (None, (FAR[1], FAR[2], 64, 1), BAD),
    (None, (FAR[0], FAR[2], 64, 2), BAD), (None, (FAR[1], FAR[1], 64, 2), BAD)])
def test_rows8_refusals(x, p, want):
    rows = sequence._ROWS.pack(*(x or (FAR[0], 64, 0)))
    kept = sequence._ROWS8.pack(*(p or (FAR[1], FAR[2], 64, 2)))
    assert abi.lib.to_rows8_pack(abi.TO_BF16, 64, 5, rows, kept, 0) == want
    assert abi.lib.to_rows8_pack(abi.TO_F64, 64, 5, rows, kept, 0) == NO
    assert abi.lib.to_rows8_unpack(abi.TO_BF16, 64, -1, kept, rows, 0) == BAD
    assert abi.lib.to_rows8_pack(abi.TO_BF16, 64, 0, rows, kept, 0) == abi.TO_OK
    assert abi.lib.to_rows8_pack(abi.TO_BF16, 64, 5, None, kept, 0) == BAD
