"""Layer norm and its gradients against 64 bits, element by element: widths from
one value to more than a workgroup holds, sizes off every vector, row strides,
rows of very different size and mean, both weight types, no rows at all.

Bounds: the statistics of a row are fp32 sums of n values, off by n 2^-24 of the
magnitudes they sum; the normalised value h inherits that relative to the row's
spread, and the mean's error relative to |mean| / sigma.
"""
import math

import numpy as np
import pytest
import torch

from decoder_ref import F, U, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def _rows(rows, n, dtype, seed, stride=None, offset=0):
    gen = torch.Generator()
    gen.manual_seed(seed)
    x = torch.randn((rows, n), generator=gen)
    x = x * (torch.rand((rows, 1), generator=gen) * 3 + 0.2) + torch.randn((rows, 1), generator=gen)
    stride = stride or n
    mem = torch.full((rows * stride + offset,), math.nan, dtype=dtype)
    mem[offset:].view(rows, stride)[:, :n] = x.to(dtype)
    return mem.cuda()[offset:].view(rows, stride)[:, :n]


class Ref:
    def __init__(self, x, w, b, eps):
        self.x = x.double()
        n = self.n = x.shape[-1]
        self.w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
        b = 0.0 if b is None else b.double()
        self.mean = self.x.mean(-1, keepdim=True)
        c = self.x - self.mean
        var = (c * c).mean(-1, keepdim=True)
        self.rstd = 1 / torch.sqrt(var + eps)
        self.h = c * self.rstd
        self.y = self.h * self.w + b
        # n values summed one after the other at worst
        self.e_mean = (n + 2) * F * self.x.abs().mean(-1, keepdim=True) + F * self.mean.abs()
        # the deviations carry the mean's error and a rounding; their squares' sum
        # is off by n + 4 roundings and by the square of the mean's error
        self.e_rstd = ((n + 8) * F + (self.e_mean * self.rstd) ** 2) * self.rstd
        self.e_h = self.e_mean * self.rstd + self.h.abs() * (self.e_rstd / self.rstd + 4 * F) \
            + F * self.x.abs() * self.rstd
        u = U[x.dtype]
        self.e_y = u * self.y.abs() + (1 + u) * (self.e_h * self.w.abs() + 2 * F * (self.y.abs() + (self.h * self.w).abs()))

    def backward(self, dy, u, uw):
        n = self.n
        dy = dy.double()
        g = dy * self.w
        m0, m1 = g.mean(-1, keepdim=True), (g * self.h).mean(-1, keepdim=True)
        dx = self.rstd * (g - m0 - self.h * m1)
        e0 = (n + 3) * F * g.abs().mean(-1, keepdim=True)
        e1 = (n + 4) * F * (g * self.h).abs().mean(-1, keepdim=True) + (g.abs() * self.e_h).mean(-1, keepdim=True)
        size = g.abs() + m0.abs() + (self.h * m1).abs()
        e = self.rstd * (e0 + self.h.abs() * e1 + self.e_h * m1.abs() + 4 * F * size) \
            + self.e_rstd * (g - m0 - self.h * m1).abs()
        rows = dy.shape[0]
        dw, db = (dy * self.h).sum(0), dy.sum(0)
        e_dw = ((rows + 4) * F * (dy * self.h).abs() + dy.abs() * self.e_h).sum(0)
        e_db = (rows + 2) * F * dy.abs().sum(0)
        tiny = 2.0**-25  # fp16 results below its normal numbers
        return ((dx, u * dx.abs() + (1 + u) * e + tiny), (dw, uw * dw.abs() + (1 + uw) * e_dw + tiny),
                (db, uw * db.abs() + (1 + uw) * e_db + tiny))


CASES = [(1, 1), (3, 2), (5, 7), (2, 64), (1, 768), (1568, 768), (33, 100), (70, 128), (9, 257), (4, 1030),
         (1100, 1030), (7, 2048), (5, 2056), (3, 8192), (2, 8200), (3, 20001), (1030, 513), (5000, 16), (2, 4096)]


@pytest.mark.parametrize("dtype,wdtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                          ("f16", "f32")])
@pytest.mark.parametrize("rows,n", CASES)
def test_against_64_bits(lc, rows, n, dtype, wdtype):
    t, wt = DTYPES[dtype], DTYPES[wdtype]
    x = _rows(rows, n, t, rows + n)
    gen = torch.Generator()
    gen.manual_seed(n)
    w = (1 + 0.3 * torch.randn(n, generator=gen)).to(wt).cuda()
    b = (0.3 * torch.randn(n, generator=gen)).to(wt).cuda()
    ref = Ref(x, w, b, 1e-5)
    print(f"[case] {rows}x{n} {dtype} {wdtype}", flush=True)
    y, mean, rstd = lc.layer_norm(x, w, b, return_stats=True)
    torch.cuda.synchronize()
    assert y.dtype == t
    assert_within(y, ref.y, ref.e_y + 2.0**-25, "y")
    assert_within(mean, ref.mean[:, 0], ref.e_mean[:, 0] + 1e-30, "mean")
    assert_within(rstd, ref.rstd[:, 0], ref.e_rstd[:, 0], "rstd")
    dy = _rows(rows, n, t, rows + n + 1)
    got = lc.layer_norm_backward(dy, x, w, mean, rstd)
    torch.cuda.synchronize()
    assert got[0].dtype == t and got[1].dtype == wt
    for name, g, (want, bound) in zip(("dx", "dweight", "dbias"), got, ref.backward(dy, U[t], U[wt])):
        assert_within(g, want, bound, name)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,stride,offset", [(96, 128, 0), (96, 97, 1), (1000, 1003, 2), (9000, 9001, 1)])
def test_row_strides(lc, dtype, n, stride, offset):
    t = DTYPES[dtype]
    x, dy = _rows(11, n, t, n, stride, offset), _rows(11, n, t, n + 1, stride + 3, offset)
    ref = Ref(x, None, None, 1e-5)
    y, mean, rstd = lc.layer_norm(x, return_stats=True)
    assert_within(y, ref.y, ref.e_y + 2.0**-25, "y")
    w = torch.ones(n, dtype=t, device="cuda")
    for g, (want, bound) in zip(lc.layer_norm_backward(dy, x, w, mean, rstd), ref.backward(dy, U[t], U[t])):
        assert_within(g, want, bound, "gradient")


def test_without_weight_and_more_dimensions(lc):
    x = _rows(24, 40, torch.float32, 1).view(2, 3, 4, 40)
    y, mean, rstd = lc.layer_norm(x, return_stats=True)
    assert y.shape == x.shape and mean.shape == (2, 3, 4)
    ref = Ref(x.reshape(24, 40), None, None, 1e-5)
    assert_within(y.view(24, 40), ref.y, ref.e_y, "y")
    dx, dw, db = lc.layer_norm_backward(x, x, None, mean, rstd)
    assert dw is None and db is None and dx.shape == x.shape
    assert_within(dx.view(24, 40), *ref.backward(x.reshape(24, 40), U[x.dtype], U[x.dtype])[0], "dx")
    assert torch.equal(lc.layer_norm(x[0, 0, 0]), y[0, 0, 0])  # one row


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_of_one_value_and_large_means(lc, dtype):
    """A constant row normalises to the bias; a mean far from zero does not eat
    the spread (fp32: 2^12 times it)."""
    t = DTYPES[dtype]
    x = torch.full((3, 300), 5.0, dtype=t, device="cuda")
    b = torch.randn(300, device="cuda").to(t)
    assert torch.equal(lc.layer_norm(x, torch.ones_like(b), b), b.expand(3, 300))
    x = _rows(6, 300, torch.float32, 5) + 4096.0
    ref = Ref(x, None, None, 1e-5)
    assert_within(lc.layer_norm(x), ref.y, ref.e_y, "y")


def test_no_rows(lc):
    x = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    y, mean, rstd = lc.layer_norm(x, w, w, return_stats=True)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = lc.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_rows_behind_the_last_stay(lc):
    mem = torch.full((10, 80), 3.0, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(10, 80, device="cuda", dtype=torch.bfloat16)
    import ctypes

    from lightning_core import _native as N
    cfg = N.LayerNormConfig(7, 80, N.LC_DTYPE_BF16, N.LC_DTYPE_BF16, 1e-5)
    st = torch.cuda.current_stream().cuda_stream
    assert N.load().lcLayerNormForward(ctypes.byref(cfg), x.data_ptr(), 80, None, None, mem.data_ptr(), 80, None, None,
                                       st) == 0
    torch.cuda.synchronize()
    assert (mem[7:] == 3).all() and torch.equal(mem[:7], lc.layer_norm(x[:7]))
    # in place
    y = lc.layer_norm(x)
    cfg = N.LayerNormConfig(10, 80, N.LC_DTYPE_BF16, N.LC_DTYPE_BF16, 1e-5)
    assert N.load().lcLayerNormForward(ctypes.byref(cfg), x.data_ptr(), 80, None, None, x.data_ptr(), 80, None, None,
                                       st) == 0
    assert torch.equal(x, y)


def test_equal_bits_and_graphs(lc):
    x, dy = _rows(700, 1000, torch.bfloat16, 1), _rows(700, 1000, torch.bfloat16, 2)
    w = torch.randn(1000, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = lc.layer_norm(x, w, w, return_stats=True)
        got = (y, mean, rstd) + tuple(lc.layer_norm_backward(dy, x, w, mean, rstd))
    for turn in range(3):
        x.copy_(_rows(700, 1000, torch.bfloat16, 10 + turn))
        graph.replay()
        y, m, r = lc.layer_norm(x, w, w, return_stats=True)
        want = (y, m, r) + tuple(lc.layer_norm_backward(dy, x, w, m, r))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_numpy_arrays(lc):
    rng = np.random.default_rng(0)
    x, dy = (rng.standard_normal((2, 5, 48)).astype(np.float32) for _ in range(2))
    w = rng.standard_normal(48).astype(np.float32)
    y, mean, rstd = lc.layer_norm(x, w, w, return_stats=True)
    got = (y, mean, rstd) + lc.layer_norm_backward(dy, x, w, mean, rstd)
    tx, tw, tdy = (torch.from_numpy(a).cuda() for a in (x, w, dy))
    ty, tm, tr = lc.layer_norm(tx, tw, tw, return_stats=True)
    want = (ty, tm, tr) + tuple(lc.layer_norm_backward(tdy, tx, tw, tm, tr))
    for a, b in zip(got, want):
        assert np.array_equal(a, b.cpu().numpy())


def test_refusals_on_the_gpu(lc):
    x = torch.randn(4, 32, device="cuda")
    with pytest.raises(ValueError, match="shape"):
        lc.layer_norm(x, torch.ones(31, device="cuda"))
    with pytest.raises(ValueError, match="type"):
        lc.layer_norm(x, torch.ones(32, device="cuda").half())
    with pytest.raises(ValueError, match="contiguous"):
        lc.layer_norm(x.t())
    with pytest.raises(ValueError, match="collapse"):
        lc.layer_norm(torch.randn(4, 3, 32, device="cuda").transpose(0, 1))
    with pytest.raises(RuntimeError, match="eps"):
        lc.layer_norm(x, eps=-1.0)
