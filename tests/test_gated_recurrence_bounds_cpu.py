"""The bounds of the recurrence's tests notice what they are there for: mistakes are planted in the 64-bit form."""
import pytest

torch = pytest.importorskip("torch")
from tests import gated_recurrence_bounds as B, recurrent_block_oracle as R  # noqa: E402


def case(tokens, channels=24):
    gen = torch.Generator().manual_seed(tokens)
    normal = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    return normal(tokens, channels), normal(tokens, channels), 1 + 7 * torch.rand(channels, generator=gen, dtype=torch.float64)


def coarse(x, f, bias, bits, every, gates=0.0):
    """h with the state rounded to `bits` at every `every` tokens, and gates off by a part `gates` of themselves."""
    a, z = torch.sigmoid(f + bias), torch.sigmoid(-(f + bias))
    a, z = torch.where(a < z, a * (1 + gates), 1 - z * (1 + gates)), torch.where(a < z, 1 - a * (1 + gates), z * (1 + gates))
    now, out = torch.zeros_like(x[0]), []
    for t in range(x.shape[0]):
        if t % every == 0:
            m, e = torch.frexp(now)
            now = torch.ldexp((m * 2 ** bits).round() / 2 ** bits, e)
        now = a[t] * now + z[t] * x[t]
        out.append(now)
    return torch.stack(out)


@pytest.mark.parametrize("tokens", [300, 2500])
def test_coarse_joins_and_gates_are_seen(tokens):
    x, f, bias = case(tokens)
    zero = torch.zeros(1, x.shape[1], dtype=torch.float64)
    h, before, _, a, z = R.recurrence(x, f, bias, [tokens], zero, True)
    bound, _ = B.values(x, f + bias, a, z, h, before, [tokens], zero, True)
    over = lambda got: float(((got - h).abs() / bound).max())  # noqa: E731
    assert over(coarse(x, f, bias, 53, 1)) < 0.01
    assert over(coarse(x, f, bias, 24, 1)) < 1  # a rounding to f32 at every token
    assert over(coarse(x, f, bias, 11, 128)) > 3  # entering states in TF32
    assert over(coarse(x, f, bias, 8, 128)) > 20  # in bf16
    assert over(coarse(x, f, bias, 53, 1, 2.0 ** -15)) > 3  # gates with 15 bits
    assert float((bound[-1] / h.abs().mean(0)).median()) < 1e-3


def test_coarse_gradients_are_seen():
    x, f, bias = case(1200)
    gen = torch.Generator().manual_seed(5)
    dh = torch.randn(1200, 24, generator=gen, dtype=torch.float64)
    zero = torch.zeros(1, 24, dtype=torch.float64)
    h, before, _, a, z = R.recurrence(x, f, bias, [1200], zero, True)
    *_, G = R.recurrence_grad(x, a, z, before, [1200], dh, zero, True)
    bound, into = B.gradients(f + bias, a, z, G, dh, zero, [1200])
    now, worst = zero[0], 0.0
    for t in range(1199, -1, -1):
        if t % 128 == 127:
            m, e = torch.frexp(now)
            now = torch.ldexp((m * 2 ** 11).round() / 2 ** 11, e)
        g = dh[t] + now
        worst, now = max(worst, float(((g - G[t]).abs() / bound[t]).max())), a[t] * g
    assert worst > 3 and ((now - a[0] * G[0]).abs() / into[0]).max() > 1
