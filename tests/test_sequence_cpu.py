"""What the sequence operators refuse, without a GPU: descriptors, sizes and
alignments are checked before anything is launched."""
import ctypes as C
import math

import pytest

from tensoroperations_b200 import abi

torch = pytest.importorskip("torch")
from tensoroperations_b200 import sequence  # noqa: E402

BOGUS = 0x1000  # an aligned address that nothing reads


def qk(**kw):
    args = dict(dtype="bf16", q_heads=4, k_heads=2, head_dim=64)
    args.update(kw)
    return sequence.QkNormRotary(**args)


@pytest.mark.parametrize("bad,status", [
    (dict(head_dim=63, rotary_dim=62), abi.TO_ERR_UNSUPPORTED), (dict(head_dim=258), abi.TO_ERR_UNSUPPORTED),
    (dict(head_dim=0, rotary_dim=0), abi.TO_ERR_UNSUPPORTED), (dict(rotary_dim=66), abi.TO_ERR_INVALID_ARGUMENT),
    (dict(rotary_dim=7), abi.TO_ERR_INVALID_ARGUMENT), (dict(sections=[16, 15]), abi.TO_ERR_INVALID_ARGUMENT),
    (dict(sections=[33, -1]), abi.TO_ERR_INVALID_ARGUMENT), (dict(q_heads=0), abi.TO_ERR_INVALID_ARGUMENT),
    (dict(k_heads=-1), abi.TO_ERR_INVALID_ARGUMENT), (dict(theta=0.0), abi.TO_ERR_INVALID_ARGUMENT),
    (dict(theta=math.inf), abi.TO_ERR_INVALID_ARGUMENT), (dict(eps=-1e-6), abi.TO_ERR_INVALID_ARGUMENT),
    (dict(eps=math.nan), abi.TO_ERR_INVALID_ARGUMENT),
])
def test_qk_plan_refusals(bad, status):
    with pytest.raises(abi.ToError) as e:
        qk(**bad)
    assert e.value.status == status


def test_python_refusals():
    with pytest.raises(ValueError):
        qk(dtype="f16")
    with pytest.raises(ValueError):
        qk(sections=[8, 8, 8, 4, 4])
    with pytest.raises(ValueError):
        sequence.LinearAttention(torch.float64, 4, 2, 64, 64)
    op = qk()
    x = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        op.forward(x, x[:, :2], None, None, None, x, x[:, :2])
    la = sequence.LinearAttention("bf16", 4, 2, 64, 64)
    with pytest.raises(ValueError, match="CUDA"):
        la.step(x, x[:, :2], x[:, :2], None, torch.zeros(3, 4, 64, 64), x)


@pytest.mark.parametrize("bad,status", [
    (dict(q_heads=4, kv_heads=3), abi.TO_ERR_INVALID_ARGUMENT), (dict(kv_heads=0), abi.TO_ERR_INVALID_ARGUMENT),
    (dict(key_dim=0), abi.TO_ERR_UNSUPPORTED), (dict(key_dim=257), abi.TO_ERR_UNSUPPORTED),
    (dict(value_dim=300), abi.TO_ERR_UNSUPPORTED), (dict(scale=math.nan), abi.TO_ERR_INVALID_ARGUMENT),
])
def test_linear_attention_refusals(bad, status):
    args = dict(dtype="f32", q_heads=4, kv_heads=2, key_dim=32, value_dim=32, scale=1.0)
    args.update(bad)
    with pytest.raises(abi.ToError) as e:
        sequence.LinearAttention(**args)
    assert e.value.status == status


def test_library_refuses_before_any_launch():
    la = sequence.LinearAttention("bf16", 4, 2, 64, 64)
    rows = (BOGUS, 4 * 64, 64)

    def args(q=rows, k=rows, v=rows, o=rows, decay=BOGUS, cu=BOGUS, slots=0, s_in=0, s_out=0):
        return sequence._ARGS.pack(*q, *k, *v, *o, decay, cu, slots, s_in, s_out, 0, 0)

    def status(fn, desc, a):
        return getattr(abi.lib, fn)(desc, a, 0)

    desc = la._desc(100, 1, 1)
    null, odd = (0, 256, 64), (BOGUS + 1, 256, 64)
    for a, want in ((args(q=null), abi.TO_ERR_INVALID_ARGUMENT), (args(k=odd), abi.TO_ERR_ALIGNMENT),
                    (args(v=(BOGUS, 32, 64)), abi.TO_ERR_INVALID_ARGUMENT), (args(o=(BOGUS, 256, 63)), abi.TO_ERR_INVALID_ARGUMENT),
                    (args(q=(BOGUS, -256, 64)), abi.TO_ERR_INVALID_ARGUMENT), (args(decay=0), abi.TO_ERR_INVALID_ARGUMENT),
                    (args(cu=0), abi.TO_ERR_INVALID_ARGUMENT), (args(cu=BOGUS + 2), abi.TO_ERR_ALIGNMENT),
                    (args(slots=BOGUS + 1), abi.TO_ERR_ALIGNMENT), (args(s_in=BOGUS + 4), abi.TO_ERR_ALIGNMENT),
                    (args(s_out=BOGUS + 8), abi.TO_ERR_ALIGNMENT)):
        assert status("to_linear_attention", desc, a) == want
    assert status("to_linear_attention", None, args()) == abi.TO_ERR_INVALID_ARGUMENT
    assert status("to_linear_attention", desc, None) == abi.TO_ERR_INVALID_ARGUMENT
    assert status("to_linear_attention", la._desc(-1, 1), args()) == abi.TO_ERR_INVALID_ARGUMENT
    assert status("to_linear_attention", la._desc(100, 70000), args()) == abi.TO_ERR_INVALID_ARGUMENT
    assert status("to_linear_attention_step", desc, args()) == abi.TO_ERR_INVALID_ARGUMENT  # no state
    assert status("to_linear_attention_step", desc, args(s_out=BOGUS + 4)) == abi.TO_ERR_ALIGNMENT
    # a long prompt needs a workspace
    assert la.workspace_bytes(100000, 1) > 0
    assert status("to_linear_attention", la._desc(100000, 1, 1), args()) == abi.TO_ERR_INVALID_ARGUMENT
    assert b"workspace" in abi.lib.to_last_error()
    grad = sequence._GRAD_ARGS.pack(*rows * 7, BOGUS, BOGUS, 0, BOGUS, BOGUS, 0, 0)
    assert status("to_linear_attention_backward", desc, grad) == abi.TO_ERR_INVALID_ARGUMENT
    assert b"dstate_in" in abi.lib.to_last_error()
    # nothing to do is not an error, whatever the pointers are
    assert status("to_linear_attention", la._desc(0, 0), args(q=null, k=null, v=null, o=null, decay=0, cu=0)) == abi.TO_OK
    assert status("to_linear_attention_step", la._desc(0, 0), args(q=null)) == abi.TO_OK


def test_workspaces_grow_with_the_work_and_say_zero_for_nothing():
    la = sequence.LinearAttention("f32", 4, 2, 64, 32)
    assert la.workspace_bytes(0, 0) == 0 and la.workspace_bytes(1, 1) == 0
    assert la.workspace_bytes(1 << 20, 1) % 256 == 0
    # gradients of shared heads pass through f32 rows of every query head
    assert la.backward_workspace_bytes(10, 1) >= 10 * 4 * (64 + 32) * 4
    assert sequence.LinearAttention("f32", 4, 4, 64, 32).backward_workspace_bytes(10, 1) == 0
    assert abi.lib.to_linear_attention_workspace_bytes(None) == 0
    assert abi.lib.to_qk_norm_rotary_workspace_bytes(None, 5) == 0


def test_null_plans():
    assert abi.lib.to_qk_plan_create(None, None) == abi.TO_ERR_INVALID_ARGUMENT
    h = C.c_void_p()
    d = abi.QkDesc(9, 4, 2, 64, 64, 1)
    assert abi.lib.to_qk_plan_create(C.byref(d), C.byref(h)) == abi.TO_ERR_UNSUPPORTED and not h.value
    r = sequence._ROWS.pack(BOGUS, 64, 64)
    assert abi.lib.to_qk_norm_rotary(None, 1, r, r, 0, 0, 0, r, r, 0) == abi.TO_ERR_INVALID_ARGUMENT
    assert abi.lib.to_qk_plan_destroy(None) == abi.TO_OK


def test_other_operators_reject_the_sequence_type():
    """TO_BF16 is known to the sequence operators alone."""
    buf = (C.c_double * 16)()
    assert abi.lib.to_synth_fill(buf, abi.TO_BF16, 4, 1, 0, 0.0, 1.0) == abi.TO_ERR_INVALID_ARGUMENT
    p = (C.c_void_p * 3)(BOGUS, BOGUS, BOGUS)
    assert abi.lib.to_sem3d_halo_pack(abi.TO_BF16, p, 0, 4, BOGUS, 0) == abi.TO_ERR_INVALID_ARGUMENT
    assert abi.lib.to_scale3(abi.TO_BF16, p, p, 4, BOGUS, 0) != abi.TO_OK
