"""Rows of the 8-bit integer operators where absolute bounds say nothing: GELU rows that lie wholly in the
negative tail, rows of a norm whose squares leave fp32's range.

GELU, u = 2^-24, exp2 and the reciprocal within one ulp (2 u).  A row of amax >= 2^-8 is x Phi(x) with Phi
from a fitted logistic form 1 / (1 + 2^w): the fit is within 3.6e-8 of Phi, w = -g(x^2) x is off by 4 u |w|
at most, which Phi (1 - Phi) |w| ln 2 <= 0.23 turns into 0.92 u, and exp2 (2 u (1 - Phi)), the sum, the
reciprocal and the product (4 u together) act on v, |v| <= |x|: |dv| <= (3.6e-8 + 0.92 u) |x| + 6 u |v| <=
(3.6e-8 + 2.92 u) |x| + 4 u |v|, whose first factor is 2.1e-7; its parts are largest at different x, and
their sum over the whole range (evaluated with every approximation at its end) stays under 0.81 of
1.6e-7 |x| + 4 u |v|, the bound that is asked for.
Rows below 2^-8 are computed relative to v: for x < -2.5 from the asymptotic form -phi(x) W(1 / x^2) with
W fitted within 5e-7, phi's exponent x^2 / 2 rounded twice with a constant (2.5 u x^2 / 2 on phi), and 12
roundings and approximate instructions of 2 u at most: |dv| <= (1e-6 + (1.25 x^2 + 24) u) |v|; elsewhere |x| <
2^-6 (v(-2.5) is above 2^-7), where Phi is 1/2 and the logistic form is off by 2 * 3.6e-8 + 8 u of v.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from test_int8_gpu import DT, D, U, _gen, _ops, _rows_check  # noqa: E402

pytestmark = pytest.mark.gpu


def _gelu_bound(x):
    """(v, dv) in 64 bits of gelu rows."""
    x = x.to(D)
    # x Phi(x) with erfc, which keeps its relative accuracy in the tail
    v = 0.5 * x * torch.special.erfc(-x * math.sqrt(0.5))
    tail = torch.where(x < -2.5, 1e-6 + (1.25 * x * x + 24) * U, torch.full_like(x, 7.2e-8 + 8 * U)) * v.abs()
    wide = 1.6e-7 * x.abs() + 4 * U * v.abs()
    # (which of the two a row within the wide bound of 2^-8 gets is the kernel's choice)
    return v, torch.where(v.abs().amax(1, keepdim=True) < 2.0 ** -8 - 1e-6, torch.minimum(tail, wide), wide)


@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", [1, 9, 384, 1000, 1531, 2999, 4096, 6145, 8192, 16384, 20001])
def test_gelu_rows_in_the_negative_tail(cols, xt):
    """Rows with no element above -2.6: their scale is a tail value."""
    m, g = _ops(), _gen(cols)
    lo = torch.tensor([2.6, 3.0, 3.1, 3.5, 4.0, 5.0, 5.5, 6.0, 7.0, 8.0, 9.0, 10.0, 10.9], device="cuda")[:, None]
    x = -(lo + (11.0 - lo) * torch.rand(13, cols, generator=g, device="cuda"))
    x[:, cols // 2] = -lo[:, 0]
    x = x.to(DT[xt])
    _rows_check(m.quantize_rows(x, act="gelu"), *_gelu_bound(x))


@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
def test_gelu_of_single_elements(xt):
    """One column: the scale is |gelu(x)| / 127 itself, over the whole range, both sides of 2^-8."""
    m = _ops()
    mag = torch.cat([torch.logspace(-4, math.log10(11.0), 1500, device="cuda"), torch.linspace(2.9, 3.2, 301, device="cuda"),
                     torch.linspace(0.0070, 0.0086, 101, device="cuda")])
    x = torch.cat([mag, -mag]).to(DT[xt])[:, None]
    r = m.quantize_rows(x, act="gelu")
    v, dv = _gelu_bound(x)
    _rows_check(r, v, dv)
    assert torch.equal(r.q[:, 0].to(torch.int32), torch.sign(v[:, 0]).to(torch.int32) * 127)


@pytest.mark.parametrize("cols", [1, 40, 700, 5000])
def test_gelu_rows_that_count_as_zeros(cols):
    """|gelu(x)| below 2^-100, zeros of both signs, padding rows; a tail beside a zero keeps its value."""
    m = _ops()
    x = torch.zeros(6, cols, device="cuda")
    x[1] = -0.0
    x[2] = -12.5
    x[3] = -60000.0
    x[4] = -3e38
    x[5, 0] = -9.0
    r = m.quantize_rows(x, act="gelu")
    assert bool((r.scale[:5] == 0).all()) and bool((r.q[:5] == 0).all())
    v = 0.5 * 9.0 * math.erfc(9.0 * math.sqrt(0.5))
    assert abs(float(r.scale[5]) * 127 / v - 1) <= 1e-6 + (1.25 * 81 + 24 + 4) * U
    assert int(r.q[5, 0]) == -127 and bool((r.q[5, 1:] == 0).all())


@pytest.mark.parametrize("cols", [1, 40, 700, 5000])
def test_gelu_rows_that_are_not_finite(cols):
    """NaN and infinities beside tail values: NaN, whichever the sign."""
    m = _ops()
    x = torch.full((4, cols), -7.0, device="cuda")
    for i, bad in enumerate((float("nan"), float("inf"), float("-inf"))):
        x[i, cols - 1] = bad
    r = m.quantize_rows(x, act="gelu")
    assert bool(r.scale[:3].isnan().all()) and bool((r.q[:3] == 0).all())
    assert bool((r.q[3] == -127).all())


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("yt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", [33, 900, 2500, 6000])
def test_norm_output_of_rows_past_fp32_is_nan(cols, yt, norm):
    """A row whose squares leave fp32's range: not only its scale but its normalised row is NaN, so that a
    residual stream does not go on from the bias; its neighbours and the stored sum are as ever."""
    m, g = _ops(), _gen(cols)
    weight = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
    bias = 0.3 * torch.randn(cols, generator=g, device="cuda")
    x = torch.randn(5, cols, generator=g, device="cuda")
    r = torch.randn(5, cols, generator=g, device="cuda")
    for b in (None, bias):
        want_y = torch.empty(5, cols, device="cuda", dtype=DT[yt])
        want = m.norm_quantize(x, weight, b, residual=r, norm=norm, eps=1e-6, norm_out=want_y)
        big = x.clone()
        big[1] *= 1e25
        big[3] = 3e38 * torch.sign(x[3])
        big[4, :] = 0.0
        big[4, cols - 1] = 1e20
        y, total = torch.zeros(5, cols, device="cuda", dtype=DT[yt]), torch.empty(5, cols, device="cuda")
        out = m.norm_quantize(big, weight, b, residual=r, norm=norm, eps=1e-6, norm_out=y, sum_out=total)
        assert bool(y[[1, 3, 4]].isnan().all())
        assert bool(out.scale[[1, 3, 4]].isnan().all()) and bool((out.q[[1, 3, 4]] == 0).all())
        assert torch.equal(total, big + r)
        assert torch.equal(y[[0, 2]], want_y[[0, 2]])
        assert torch.equal(out.q[[0, 2]], want.q[[0, 2]]) and torch.equal(out.scale[[0, 2]], want.scale[[0, 2]])
