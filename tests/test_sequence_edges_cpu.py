"""What the sequence operators refuse of memory that is read and written in one call, without a
GPU: the addresses are checked before anything is launched."""
import pytest

from tensoroperations_b200 import abi

pytest.importorskip("torch")
from tensoroperations_b200 import sequence  # noqa: E402

FAR = 1 << 24
AT = [FAR * (i + 1) for i in range(8)]  # aligned addresses far apart, which nothing reads
LIST = 16 * FAR                         # one for the lists
T, HQ, HK, D = 100, 4, 2, 64


def refused(status, *words):
    text = abi.lib.to_last_error().decode()
    return status == abi.TO_ERR_INVALID_ARGUMENT and "share memory" in text and all(w in text for w in words)


def rows(at, heads):
    return at, heads * D, D


# another tensor's address: the same, some rows on, and one value before its end
SHIFTS = [0, 2 * D, 2 * 3 * D, 2 * (T * HK * D - 1)]


@pytest.mark.parametrize("shift", SHIFTS)
@pytest.mark.parametrize("call", ["to_linear_attention", "to_linear_attention_step"])
@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_outputs_are_not_what_is_read(call, name, shift):
    la = sequence.LinearAttention("bf16", HQ, HK, D, D)
    at = dict(q=rows(AT[0], HQ), k=rows(AT[1], HK), v=rows(AT[2], HK))
    o = (at[name][0] + shift, *at[name][1:]) if name == "q" else (at[name][0] + shift, HQ * D, D)
    args = sequence._ARGS.pack(*at["q"], *at["k"], *at["v"], *o, LIST, LIST, 0, 0, AT[5], 0, 0)
    if name != "q" and shift:  # token strides differ: only ranges are known, which may pass
        return
    assert refused(getattr(abi.lib, call)(la._desc(T, 1, T), args, 0), "o", name)


@pytest.mark.parametrize("shift", [4 * HQ * D * D, -4 * HQ * D * D, 16])
def test_states_overlap_whole_or_not_at_all(shift):
    la = sequence.LinearAttention("bf16", HQ, HK, D, D)
    r = rows(AT[0], HQ), rows(AT[1], HK), rows(AT[2], HK), rows(AT[3], HQ)
    args = sequence._ARGS.pack(*r[0], *r[1], *r[2], *r[3], LIST, LIST, 0, AT[5], AT[5] + shift, 0, 0)
    assert refused(abi.lib.to_linear_attention(la._desc(T, 3, 3), args, 0), "state_in", "state_out")
    args = sequence._ARGS.pack(*r[0], *r[1], *r[2], *r[3], LIST, LIST, LIST, AT[5], AT[5] + shift, 0, 0)
    assert refused(abi.lib.to_linear_attention(la._desc(T, 1, 5), args, 0), "state_in", "state_out")


GRAD = ["q", "k", "v", "d_o", "dq", "dk", "dv"]


def gradient_status(heads_k=HK, state_in=0, dstate_out=0, dstate_in=0, **moved):
    la = sequence.LinearAttention("bf16", HQ, heads_k, D, D)
    at = {n: rows(AT[i], HQ if n in ("q", "d_o", "dq") else heads_k) for i, n in enumerate(GRAD)}
    at.update(moved)
    args = sequence._GRAD_ARGS.pack(*(x for n in GRAD for x in at[n]), LIST, LIST, state_in, dstate_out, dstate_in,
                                    1 << 40, 1 << 30)  # (a workspace)
    return abi.lib.to_linear_attention_backward(la._desc(T, 3, 3), args, 0)


@pytest.mark.parametrize("shift", SHIFTS)
@pytest.mark.parametrize("out", ["dq", "dk", "dv"])
def test_gradients_are_not_what_is_read(out, shift):
    for other in GRAD:
        if other != out:
            status = gradient_status(heads_k=HQ, **{out: rows(AT[GRAD.index(other)] + shift, HQ)})
            assert refused(status, out, other), (out, other, abi.lib.to_last_error())


@pytest.mark.parametrize("name", ["state_in", "dstate_out"])
def test_state_gradients_are_not_what_is_read(name):
    for shift in (0, 16, 4 * HQ * D * D):
        assert refused(gradient_status(dstate_in=AT[7] + shift, **{name: AT[7]}), "dstate_in", name)


def test_rows_of_an_output_lie_apart():
    # tokens that begin inside the last one's heads; heads inside one another's tokens
    for layout in ((D, D), (2 * D + D // 2, D), (D, 3 * D)):
        assert refused(gradient_status(dq=(AT[4], *layout)), "dq"), layout
        la = sequence.LinearAttention("bf16", HQ, HK, D, D)
        args = sequence._ARGS.pack(*rows(AT[0], HQ), *rows(AT[1], HK), *rows(AT[2], HK), AT[3], *layout, LIST, LIST, 0, 0,
                                   AT[5], 0, 0)
        assert refused(abi.lib.to_linear_attention_step(la._desc(T, 0, T), args, 0), "o"), layout


@pytest.mark.parametrize("backward", [False, True])
def test_norm_and_rotation_outputs(backward):
    op = sequence.QkNormRotary("bf16", HQ, HQ, D)
    names = ["q", "k", "gq", "gk", "dq", "dk"] if backward else ["q", "k", "q_out", "k_out"]

    def status(**moved):
        at = {n: rows(AT[i], HQ) for i, n in enumerate(names)}
        at.update(moved)
        r = [sequence._ROWS.pack(*at[n]) for n in names]
        if backward:
            return abi.lib.to_qk_norm_rotary_backward(op._h, T, r[0], r[1], LIST, 0, 0, *r[2:], 0, 0, LIST, 1 << 30, 0)
        return abi.lib.to_qk_norm_rotary(op._h, T, r[0], r[1], LIST, 0, 0, *r[2:], 0)

    for out in names[-2:]:
        for other in names:
            if other != out:
                at = AT[names.index(other)]
                own = other.strip("dg_out") == out.strip("dg_out")
                if not own:  # in place is a head's own rows
                    assert refused(status(**{out: rows(at, HQ)}), out, other)
                assert refused(status(**{out: rows(at + 2 * D, HQ)}), out, other)
                assert refused(status(**{out: (at, 2 * HQ * D, D)}), out, other)  # other strides
        assert refused(status(**{out: (AT[7], D, D)}), out)


@pytest.mark.parametrize("bad", [dict(q_heads=2**32 + 4), dict(k_heads=2**32), dict(head_dim=2**32 + 64),
                                 dict(rotary_dim=2**32 + 64), dict(sections=[2**32 + 32]), dict(q_heads=-2**32 + 4)])
def test_sizes_past_32_bits_are_not_cut_short(bad):
    args = dict(dtype="bf16", q_heads=4, k_heads=2, head_dim=64)
    args.update(bad)
    with pytest.raises((ValueError, abi.ToError)):
        sequence.QkNormRotary(**args)
    args = {n: v for n, v in args.items() if n in ("dtype", "q_heads")}
    if "q_heads" in bad:
        with pytest.raises((ValueError, abi.ToError)):
            sequence.LinearAttention(**args, kv_heads=2, key_dim=64, value_dim=64)


@pytest.mark.parametrize("key_dim", [0, -4, 2**32 + 64])
def test_key_widths_are_refused_before_their_root_is_taken(key_dim):
    with pytest.raises((ValueError, abi.ToError)):
        sequence.LinearAttention("f32", 4, 2, key_dim, 32)
