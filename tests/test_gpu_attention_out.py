"""The output tensor that a caller hands to cross attention."""
import pytest
import torch

from gpu_util import require_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def test_keys_and_values_are_not_overwritten(lc):
    q, k, v = (torch.randn(1, 2, 9, 64, device="cuda") for _ in range(3))
    for x in (k, v):
        before = x.clone()
        with pytest.raises(ValueError, match="out must not be k or v"):
            lc.cross_attention(q, k, v, out=x)
        assert torch.equal(x, before)
    a, b = k.cpu().numpy(), v.cpu().numpy()
    with pytest.raises(ValueError, match="out must not be k or v"):
        lc.cross_attention(q.cpu().numpy(), a, b, out=a)


@pytest.mark.parametrize("sq,sk", [(9, 9), (3, 5000), (1500, 300)])
def test_out_may_be_q(lc, sq, sk):
    """A workgroup reads its query rows before it writes them, and no other reads them."""
    q, k, v = (torch.randn(4, 8, s, 64, device="cuda", dtype=torch.bfloat16) for s in (sq, sk, sk))
    want = lc.cross_attention(q, k, v)
    assert lc.cross_attention(q, k, v, out=q) is q
    assert torch.equal(q, want)


def test_an_out_whose_heads_overlap_is_refused(lc):
    q, k = torch.randn(2, 2, 3, 64, device="cuda"), torch.randn(2, 2, 9, 64, device="cuda")
    mem = torch.zeros(1000, device="cuda")
    for strides in ((64, 64, 128, 1), (192, 192, 64, 1), (128, 192, 64, 1)):
        with pytest.raises(RuntimeError, match="overlapping rows"):
            lc.cross_attention(q, k, k, out=mem.as_strided((2, 2, 3, 64), strides))
    assert (mem == 0).all()
    out = mem.as_strided((2, 2, 3, 64), (64, 384, 128, 1))
    lc.cross_attention(q, k, k, out=out)
    assert torch.equal(out, lc.cross_attention(q, k, k))
