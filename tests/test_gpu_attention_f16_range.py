"""fp16 cross attention where its second operands leave fp16's range: gradients of
values far from one, and of keys so many that each has a probability far below
the normal numbers.  Whatever the operands' size, a result that fp16 can hold has
fp16's precision.
"""
import math

import pytest
import torch

from decoder_ref import F, U, Attention, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu

HALF = torch.float16
STEP = U[HALF]


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def _randn(shape, seed):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return torch.randn(shape, generator=gen)


def _gradients(lc, q, k, v, dout, lengths, what):
    print(f"[case] {what}", flush=True)
    ref = Attention(q, k, v, lengths)
    out, lse = lc.cross_attention(q, k, v, lengths, return_lse=True)
    got = lc.cross_attention_backward(dout, q, k, v, out, lse, lengths)
    torch.cuda.synchronize()
    for name, x in zip(("dq", "dk", "dv"), got):
        want, bound = ref.backward(dout)[name]
        assert want.abs().max() < 60000, "the case is to stay inside fp16"
        assert_within(x, want, bound, f"{what} {name}")


@pytest.mark.parametrize("padded", [2, 700])
def test_two_keys_far_apart(lc, padded):
    """dO = 1 over 128 values of 20000 and of 0: dS is 640000, dQ 11314."""
    q = (_randn((1, 2, 40, 128), 1) * 0.01).to(HALF).cuda()
    k = torch.full((1, 2, padded, 128), math.nan, dtype=HALF)
    v = torch.full_like(k, math.nan)
    k[:, :, 0], k[:, :, 1] = 0.1, -0.1
    v[:, :, 0], v[:, :, 1] = 20000, 0
    dout = torch.ones((1, 2, 40, 128), dtype=HALF, device="cuda")
    lengths = torch.tensor([2], dtype=torch.int32, device="cuda")
    _gradients(lc, q, k.cuda(), v.cuda(), dout, lengths, f"two keys, padded to {padded}")


@pytest.mark.parametrize("sq,sk", [(33, 5), (300, 40), (70, 300)])
def test_large_values_and_gradients_of_every_size(lc, sq, sk):
    """Values of 8000, rows of dO from 2^-14 to 2^4 and one of zeros, in an order
    that moves the scale up and down from row to row and from key to key."""
    q = (_randn((2, 2, sq, 64), 2) * 0.3).to(HALF).cuda()
    k = (_randn((2, 1, sk, 64), 3) * 0.05).to(HALF).cuda()
    v = (_randn((2, 1, sk, 64), 4) * 8000).clamp(-30000, 30000)
    v[:, :, ::3] *= 2.0**-12
    v[:, :, 1::4] *= -1
    dout = _randn((2, 2, sq, 64), 5) * 2.0 ** ((torch.arange(sq) * 7) % 19 - 14).view(1, 1, sq, 1)
    dout[:, :, 2] = 0
    dout = dout * 2.0**-6  # what keeps the sums over all rows inside fp16
    _gradients(lc, q, k, v.to(HALF).cuda(), dout.to(HALF).cuda(), None, f"large values {sq}x{sk}")


def _many_keys(lc):
    """Keys of equal probability, so many that P is 64.5 steps of fp16's
    subnormal numbers; gradients in which every key counts with the same sign.

    Columns: 0 carries dP (V = +-1, dO = 1) and dQ (K = +-1/2); 1 carries dK (Q =
    8, K = 0), so that all scores are zero.  delta is zero.
    """
    rows, keys, d = 64, 260_112, 64
    sign = 1.0 - 2.0 * (torch.arange(keys) % 2)
    q, dout = torch.zeros((1, 1, rows, d)), torch.zeros((1, 1, rows, d))
    k, v = torch.zeros((1, 1, keys, d)), torch.zeros((1, 1, keys, d))
    q[..., 1], dout[..., 0] = 8.0, 1.0
    k[..., 0], v[..., 0] = 0.5 * sign, sign
    q, k, v, dout = (x.to(HALF).cuda() for x in (q, k, v, dout))
    lse = torch.full((1, 1, rows), math.log(keys), dtype=torch.float32, device="cuda")
    print("[case] many keys", flush=True)
    got = lc.cross_attention_backward(dout, q, k, v, torch.zeros_like(q), lse)
    torch.cuda.synchronize()
    sign = sign.double().cuda()
    scale, p = d**-0.5, 1.0 / keys
    want = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in got]
    want[0][..., 0] = 0.5 * scale
    want[1][..., 1] = sign * (rows * 8.0 * p * scale)
    want[2][..., 0] = rows * p
    return got, want, rows, keys


# lse is a rounded 12.5, so P is off by 12.5 2^-24 and the exponential's own error.
E_P = 16 * F


def test_many_keys_dq(lc):
    """The products run over the keys, 16 to an instruction: at worst two
    roundings of the sum for each."""
    got, want, _, keys = _many_keys(lc)
    bound = want[0].abs() * (2 * STEP + E_P + keys / 8 * F) * 1.01
    assert_within(got[0], want[0], bound + 2.0**-25, "dq")


def test_many_keys_dk(lc):
    got, want, rows, _ = _many_keys(lc)
    bound = want[1].abs() * (2 * STEP + E_P + rows * F) * 1.01
    assert_within(got[1], want[1], bound + 2.0**-25, "dk")


def test_many_keys_dv(lc):
    got, want, rows, _ = _many_keys(lc)
    bound = want[2].abs() * (2 * STEP + E_P + rows * F) * 1.01
    assert_within(got[2], want[2], bound + 2.0**-25, "dv")


@pytest.mark.parametrize("rows,score", [(3, 11.75), (65536, 14.25)])
def test_many_keys_far_below_one(lc, rows, score):
    """One key whose score is far above those of 65536 equal ones: half of the
    columns are theirs alone.  Few rows: each wave has some of the keys; many: all."""
    keys, d = 65537, 64
    q, k, v = (torch.zeros((1, 1, n, d)) for n in (rows, keys, keys))
    q[..., 0], k[..., 0, 0] = 8.0, score
    v[..., 1:, :32], v[..., 0, 32:] = 1.0, 1.0
    q, k, v = (x.to(HALF).cuda() for x in (q, k, v))
    print("[case] one key above many", flush=True)
    out, lse = lc.cross_attention(q, k, v, return_lse=True)
    torch.cuda.synchronize()
    rest = (keys - 1) * math.exp(-score)
    total = 1 + rest
    want = torch.full(out.shape, 1 / total, dtype=torch.float64, device="cuda")
    want[..., :32] = rest / total
    # P and the result rounded to fp16; the score in exp2 units and the
    # exponential.  A lane adds up at most half the keys for l, and a wave's
    # products all of them, 16 to an instruction with at most two roundings.
    e_sum = (keys / 2 + keys / 8 + 64) * F
    assert_within(out, want, want * (2 * STEP + e_sum) * 1.01, "out")
    assert_within(lse, torch.full(lse.shape, score + math.log(total), dtype=torch.float64, device="cuda"),
                  torch.full(lse.shape, e_sum, dtype=torch.float64, device="cuda"), "lse")
