"""The gradient of a layer norm's bias where the norm has no weight."""
import numpy as np
import pytest
import torch

from gpu_util import require_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc():
    return require_hip()


@pytest.mark.parametrize("dtype,btype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                         (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,n", [(0, 40), (1, 7), (300, 96), (50, 1030), (5, 9000)])
def test_bias_alone(lc, rows, n, dtype, btype):
    gen = torch.Generator()
    gen.manual_seed(rows + n)
    x, dy = (torch.randn((rows, n), generator=gen).to(dtype).cuda() for _ in range(2))
    b = torch.randn(n, generator=gen).to(btype).cuda()
    y, mean, rstd = lc.layer_norm(x, None, b, return_stats=True)
    dx, dw, db = lc.layer_norm_backward(dy, x, None, mean, rstd, bias=b)
    assert dw is None and db.dtype == btype and db.shape == (n,)
    # the same sums as beside a weight of ones, and the same dx
    ones = torch.ones(n, dtype=btype, device="cuda")
    dx1, _, db1 = lc.layer_norm_backward(dy, x, ones, mean, rstd)
    assert torch.equal(db, db1) and torch.equal(dx, dx1)
    assert torch.equal(dx, lc.layer_norm_backward(dy, x, None, mean, rstd)[0])
    # with both, the bias changes nothing
    assert torch.equal(db, lc.layer_norm_backward(dy, x, ones, mean, rstd, bias=b)[2])


def test_numpy_and_refusals(lc):
    x = np.random.default_rng(1).standard_normal((6, 20)).astype(np.float32)
    b = np.zeros(20, np.float32)
    y, mean, rstd = lc.layer_norm(x, None, b, return_stats=True)
    dx, dw, db = lc.layer_norm_backward(x, x, None, mean, rstd, bias=b)
    assert dw is None and np.allclose(db, x.sum(0), rtol=0, atol=8 * 2.0**-24 * np.abs(x).sum(0).max())
    with pytest.raises(ValueError, match="bias has shape"):
        lc.layer_norm_backward(x, x, None, mean, rstd, bias=b[:19])
    with pytest.raises(ValueError, match="one type"):
        h = x.astype(np.float16)
        lc.layer_norm_backward(h, h, np.ones(20, np.float16), mean, rstd, bias=b)
