"""The tolerances of the block-scaled product, on the host: what they accept and which mistakes they reject at the head's sizes."""

import pytest

torch = pytest.importorskip("torch")

from tests import head_sums  # noqa: E402

E4M3 = torch.float8_e4m3fn


def operands(rows, units, inner):
    g = torch.Generator().manual_seed(rows + units + inner)
    a = torch.randn((rows, inner), generator=g).clamp_min(-0.3)
    b = torch.randn((units, inner), generator=g)
    across = -(-inner // 128)
    sa = torch.exp2(torch.randn((rows, across), generator=g))
    sb = torch.exp2(torch.randn((-(-units // 128), across), generator=g)) * 2.0 ** -16
    return (a * 80).clamp(-448, 448).to(E4M3), sa, (b * 80).clamp(-448, 448).to(E4M3), sb


def cut(a, sa, b, sb):
    """The sums with each product cut below 2^-13 of the largest of its eight, by the exponents."""
    x, w = a.float().double(), b.float().double()
    inner = x.shape[1]
    power = lambda v: torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))  # noqa: E731
    y = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64)
    for k in range(0, inner, 8):
        p = x[:, None, k:k + 8] * w[None, :, k:k + 8]
        step = torch.exp2((power(x)[:, None, k:k + 8] + power(w)[None, :, k:k + 8]).amax(2, keepdim=True) - 13)
        y += (torch.trunc(p / step) * step).sum(2) * sa[:, k // 128, None].double() * sb[0, k // 128].double()
    return y


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_tolerance_rejects_what_it_should(dtype):
    rows, units, inner = 12, 96, 28224
    a, sa, b, sb = operands(rows, units, inner)
    y, l2 = head_sums.product(a, sa, b, sb)
    narrow = dtype != torch.float32
    allowed = head_sums.tolerance(y, l2, inner, dtype, narrow)
    accepted = lambda got: bool(((got.to(dtype).double() - y).abs() <= allowed).all())  # noqa: E731
    assert accepted(y)
    x, w = head_sums.dequantized(a, sa, 1), head_sums.dequantized(b, sb, 128)
    # a sum in fp32, one product after the other in 64 lanes
    lanes = torch.zeros((64, rows, units))
    for k in range(0, inner, 64):
        lanes += (x[:, k:k + 64].t()[:, :, None] * w[:, k:k + 64].t()[:, None, :]).float()
    assert accepted(lanes.sum(0))
    if narrow:
        some = (slice(0, 3), slice(0, 24))
        assert ((cut(a[some[0]], sa[some[0]], b[some[1]], sb).to(dtype).double() - y[some]).abs() <= allowed[some]).all()
    part = lambda s: x[:, s] @ w[:, s].t()  # noqa: E731
    for what, got in {"a chunk of 16 bytes lost": y - part(slice(27008, 27024)), "a chunk counted twice": y + part(slice(128, 144)),
                      "a block lost": y - part(slice(6400, 6528)), "the partial block lost": y - part(slice(28160, inner)),
                      "a wrong scale": y - 0.4 * part(slice(19200, 19328)), "all scaled": y * 1.005,
                      "one row's first block lost": y - torch.where(torch.arange(rows)[:, None] == 3, part(slice(0, 128)), 0.0)}.items():
        assert not accepted(got), what
