"""Layer norm of fp32 rows whose mean is far above their spread: the statistics
are as good as the spread allows, not as the mean's magnitude does.

A thread sums at most 36 values one after the other and ten joins follow (n <=
9000), so a sum is off by at most DEPTH 2^-24 of the magnitudes it holds.
"""
import pytest
import torch

from decoder_ref import F, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu

DEPTH = 48
WIDTHS = [3, 100, 300, 768, 1030, 2056, 8192, 8200, 9000]


@pytest.fixture(scope="module")
def lc():
    return require_hip()


@pytest.mark.parametrize("n", WIDTHS)
def test_constant_rows(lc, n):
    """Every deviation is zero: y is the bias, the mean the constant itself."""
    values = torch.tensor([10000.1, 1000.1, 30000.7, 0.1, -1 / 3, 7e-5, 123456.7, 1e20, 5.0, 0.0])
    x = values.view(-1, 1).expand(-1, n).contiguous().cuda()
    w, b = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    for rows in (x, x.repeat(130, 1)):  # few rows: a workgroup each; many: a wave
        y, mean, rstd = lc.layer_norm(rows, w, b, return_stats=True)
        assert torch.equal(y, b.expand_as(y))
        assert torch.equal(mean, rows[:, 0].contiguous())
        want = torch.full((len(rows),), 1e-5**-0.5, dtype=torch.float64, device="cuda")
        assert_within(rstd, want, want * 4 * F, "rstd")
        dy = torch.randn_like(rows)
        dx, dw, db = lc.layer_norm_backward(dy, rows, w, mean, rstd)
        assert (dw == 0).all()
        g = dy.double() * w.double()
        centred = (g - g.mean(-1, keepdim=True)) * want.view(-1, 1)
        size = (g.abs() + g.abs().mean(-1, keepdim=True) * DEPTH) * want.view(-1, 1)
        assert_within(dx, centred, size * 8 * F, "dx")


@pytest.mark.parametrize("n", WIDTHS[1:])
@pytest.mark.parametrize("mean,spread", [(10000.1, 0.01), (-300.3, 1e-3), (30000.7, 1.0), (1.0, 1e-6)])
def test_spread_far_below_the_mean(lc, n, mean, spread):
    gen = torch.Generator()
    gen.manual_seed(n)
    x = (mean + spread * torch.randn((40, n), generator=gen, dtype=torch.float64)).float().cuda()
    eps = 1e-3 * spread**2
    y, mu, rstd = lc.layer_norm(x, eps=eps, return_stats=True)
    xd = x.double()
    m = xd.mean(-1, keepdim=True)
    c = xd - m
    var = (c * c).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + float(torch.tensor(eps, dtype=torch.float32)))
    # the first mean is off by `first`; x less that mean is exact or rounds once,
    # and the deviations' own sum is off by DEPTH roundings of their size
    first = DEPTH * F * xd.abs().mean(-1, keepdim=True)
    e_off = (DEPTH + 2) * F * (c.abs().mean(-1, keepdim=True) + first)
    e_c = e_off + 3 * F * (c.abs() + first)
    # squares about the first mean, less that mean's own square
    e_var = (DEPTH + 6) * F * (var + 2 * first**2) + 2 * first * e_off
    e_rel = 0.5 * e_var * r * r + 4 * F
    bound = e_c * r + (c * r).abs() * (e_rel + 4 * F)
    assert_within(y, c * r, bound * 1.01, "y")
    assert_within(mu.view(-1, 1), m, e_off + F * m.abs(), "mean")
    assert_within(rstd.view(-1, 1), r, r * e_rel * 1.01, "rstd")
