"""Gradients of the norms around a block for rows at the ends of the range, against plain 64-bit forms."""
import pytest

torch = pytest.importorskip("torch")
from tensoroperations_b200 import sequence  # noqa: E402
from tests import recurrent_block_oracle as R  # noqa: E402
from tests.recurrent_block_oracle import U, d  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def close(got, want, tol, what):
    got, want = d(got), d(want)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - tol
    assert over.max() <= 0, f"{what}: {over.max():.3g} over the bound, relative error {((got - want).abs() / want.abs()).max():.3g}"


def gradients(op, dtype, residual, r, y, dro, dn, w_pre, w_post):
    tokens, width = r.shape
    dr, dy = torch.empty_like(r), torch.empty_like(y)
    dw_post, dw_pre = (torch.empty(width, device="cuda") for _ in "ab")
    ws = torch.empty(op.workspace_bytes(tokens), dtype=torch.uint8, device="cuda")
    op.backward(r, y, None, w_post, w_pre, dro, dn, dr, dy, None, dw_post, dw_pre, ws)
    return dr, dy, dw_pre, dw_post


@pytest.mark.parametrize("dtype,residual", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("width", [264, 1003])
@pytest.mark.parametrize("size,eps", [(1e-14, 0.0), (1e-17, 0.0), (1e-6, 0.0), (1e13, 1e-6), (1e15, 1e-6), (1e17, 0.0)])
def test_gradients_of_small_and_large_rows(dtype, residual, width, size, eps):
    """The stream's rows are `size` large; dr is then of order 1 / size, far from where 1 / rms^3 has left f32."""
    gen = torch.Generator("cuda").manual_seed(width)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    r, y, dn = (size * normal(21, width)).to(residual), normal(21, width).to(dtype), normal(21, width).to(dtype)
    dn = (dn.float() + r.float() / size).to(dtype)  # so that the part along r is as large as the others
    w_pre, w_post = 1 + 0.3 * normal(width), 1 + 0.3 * normal(width)
    op = sequence.BlockNorm(dtype, width, residual=residual, scale=0.5, eps=eps)
    dr, dy, dw_pre, dw_post = gradients(op, dtype, residual, r, y, None, dn, w_pre, w_post)
    r0, y0, dn0, p0, n0 = d(r), d(y), d(dn), d(w_post), d(w_pre)
    pr, py = R.rms(r0, eps), R.rms(y0, eps)
    # sums of `width` terms: 32 additions in a row at most, and the products and roots around them
    count = 64 * U
    e, rh = n0 * dn0, r0 / pr
    along = (e * rh).mean(-1, keepdim=True)
    t = (e - rh * along) / pr
    tt = 2 * count * (e.abs() + rh.abs() * (e * rh).abs().mean(-1, keepdim=True)) / pr
    close(dr, t, tt + R.rounding(residual) * t.abs(), "dr")
    close(dw_pre, (dn0 * rh).sum(0), (21 + 64) * U * (dn0 * rh).abs().sum(0), "dw_pre")
    q, yh = 0.5 * t, y0 / py
    tu = 0.5 * tt + count * q.abs()
    close(dw_post, (q * yh).sum(0), ((21 + 64) * U * (q * yh).abs() + tu * yh.abs()).sum(0), "dw_post")
    e, te = p0 * q, p0.abs() * tu
    wy = (e - yh * (e * yh).mean(-1, keepdim=True)) / py
    ty = (te + yh.abs() * ((te + 2 * count * e.abs()) * yh.abs()).mean(-1, keepdim=True)) / py + \
        2 * count * (e.abs() + yh.abs() * (e * yh).abs().mean(-1, keepdim=True)) / py
    close(dy, wy, ty + R.rounding(dtype) * wy.abs(), "dy")


@pytest.mark.parametrize("dtype,residual", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_a_padding_row_with_a_small_eps_spoils_nothing(dtype, residual):
    """A row of zeros (dr = w dn / sqrt(eps)) among others: finite, and no NaN in the sums over the rows."""
    gen = torch.Generator("cuda").manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    r, y, dn = normal(9, 320).to(residual), normal(9, 320).to(dtype), normal(9, 320).to(dtype)
    r[4] = 0
    w = 1 + 0.3 * normal(320)
    op = sequence.BlockNorm(dtype, 320, residual=residual, eps=1e-30)
    dr, dy, dw_pre, dw_post = gradients(op, dtype, residual, r, y, None, dn, w, None)
    assert all(torch.isfinite(t).all() for t in (dr, dy, dw_pre, dw_post))
    want = d(w) * d(dn)[4] * 1e15
    close(dr[4], want, (R.rounding(residual) + 8 * U) * want.abs(), "dr")
