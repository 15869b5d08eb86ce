"""The decoder operators as they are used together: an image through the ViT
block, its tokens through layer norm and cross attention with gradients, and the
same tokens through the 8-bit cache token by token.
"""
import math

import numpy as np
import pytest
import torch

from decoder_ref import Attention, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def _vit_weights(rng, embed, patch):
    return (rng.standard_normal((embed, 3, patch, patch)).astype(np.float32) * np.float32((3 * patch**2) ** -0.5),
            rng.standard_normal((embed, 3 * embed)).astype(np.float32) * np.float32(embed**-0.5),
            rng.standard_normal((embed, embed)).astype(np.float32) * np.float32(embed**-0.5))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_vit_block_with_a_norm(lc, dtype):
    """The block's norm against its definition in fp64 on the block's own roundings."""
    rng = np.random.default_rng(4)
    embed, heads, patch = 256, 4, 16
    w_conv, w_qkv, w_o = _vit_weights(rng, embed, patch)
    x = rng.standard_normal((2, 3, 64, 96)).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(embed)).astype(np.float32)
    b = (0.2 * rng.standard_normal(embed)).astype(np.float32)
    s = lc.VitBlockSession(2, 3, 64, 96, patch, embed, heads, dtype)
    s.set_weights(w_conv, w_qkv, w_o)
    plain = s.forward(x)
    s.set_norm(w, b, 1e-5)
    got = s.forward(x)
    s.run_cached(2)
    assert np.array_equal(s.forward(), got)
    s.set_norm(None)
    assert np.array_equal(s.forward(), plain)
    s.close()
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]

    def r(a):
        return torch.as_tensor(np.asarray(a)).to(t).double()

    def rt(a):
        return a.to(t).double()

    patches = r(x).unfold(2, patch, patch).unfold(3, patch, patch).permute(0, 2, 3, 1, 4, 5).reshape(2, 24, -1)
    tokens = rt(torch.relu(patches @ r(w_conv).reshape(embed, -1).t()))
    c = tokens - tokens.mean(-1, keepdim=True)
    tokens = rt(c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * torch.from_numpy(w).double()
                + torch.from_numpy(b).double())
    q, k, v = rt(tokens @ r(w_qkv)).view(2, 24, 3, heads, 64).permute(2, 0, 3, 1, 4)
    p = torch.softmax(q @ k.transpose(-1, -2) / 8, -1)
    want = rt((p @ v).permute(0, 2, 1, 3).reshape(2, 24, embed)) @ r(w_o)
    got = torch.from_numpy(got).double()
    # tokens, norm, q / k / v and attention output are each rounded to the type,
    # and a value next to a border may fall on its other side: four steps
    step = {"bf16": 2.0**-7, "f16": 2.0**-10}[dtype]
    assert ((got - want).norm(dim=-1) <= 4 * step * want.norm(dim=-1)).all()


def test_image_to_decoder_and_back(lc):
    rng = np.random.default_rng(5)
    embed, heads, batch = 256, 4, 3
    s = lc.VitBlockSession(batch, 3, 64, 64, 8, embed, heads, "bf16")
    s.set_weights(*_vit_weights(rng, embed, 8))
    s.set_norm(np.ones(embed))
    states = torch.from_numpy(s.forward(rng.standard_normal((batch, 3, 64, 64)).astype(np.float32))).cuda()
    s.close()
    tokens = states.shape[1]
    t = torch.bfloat16
    gen = torch.Generator()
    gen.manual_seed(6)
    lengths = torch.tensor([tokens, 40, 0], dtype=torch.int32, device="cuda")
    x = torch.randn((batch, 19, embed), generator=gen).to(t).cuda()
    w = (1 + 0.1 * torch.randn(embed, generator=gen)).cuda()
    b = (0.1 * torch.randn(embed, generator=gen)).cuda()

    def split(y):
        return y.view(batch, -1, heads, embed // heads).transpose(1, 2)

    # forward: norm of the decoder's rows, then attention to the image's states
    n, mean, rstd = lc.layer_norm(x, w, b, return_stats=True)
    q, kv = split(n), split(states.to(t))
    out, lse = lc.cross_attention(q, kv, kv, lengths, return_lse=True)
    # backward of sum(out * g) to x, the weights and the states
    g = torch.randn((batch, 19, embed), generator=gen).to(t).cuda()
    dq, dk, dv = lc.cross_attention_backward(split(g), q, kv, kv, out, lse, lengths)
    dn = dq.transpose(1, 2).reshape(batch, 19, embed)
    dx, dw, db = lc.layer_norm_backward(dn, x, w, mean, rstd)

    # the same in 64 bits with autograd, from the unrounded norm
    leaves = [y.double().requires_grad_() for y in (x, w, b, states.to(t))]
    lx, lw, lb, ls = leaves
    ln = torch.nn.functional.layer_norm(lx, (embed,), lw, lb, 1e-5)
    lq, lkv = split(ln), split(ls)
    sc = lq @ lkv.transpose(-1, -2) / math.sqrt(embed // heads)
    hidden = torch.arange(tokens, device="cuda") >= lengths.view(-1, 1, 1, 1)
    lout = torch.softmax(sc[:2].masked_fill(hidden[:2], -math.inf), -1) @ lkv[:2]
    (lout * split(g)[:2].double()).sum().backward()
    assert (out[2] == 0).all() and (dq[2] == 0).all() and (dk[2] == 0).all() and (dv[2] == 0).all()
    u = 2.0**-8
    for name, got, want, steps in (
            ("out", out[:2], lout, 3),          # norm, probabilities, result
            ("dstates", (dk + dv).transpose(1, 2).reshape(states.shape), ls.grad, 6),
            ("dx", dx[:2], lx.grad[:2], 8),     # and dq, dS, delta, dn, dx
            ("dweight", dw, lw.grad, 8), ("dbias", db, lb.grad, 8)):
        off = (got.double() - want).norm() / want.norm()
        print(f"[parity] {name}: {off:.3e} of {steps * u:.3e}", flush=True)
        assert off <= steps * u, name


def test_decode_over_the_cache_follows_the_whole_attention(lc):
    """Token by token over the cache against one attention over the values that
    the cache holds."""
    gen = torch.Generator()
    gen.manual_seed(7)
    b, heads, d, sk = 2, 4, 64, 150
    t = torch.float16
    states = torch.randn((b, sk, 2, heads, d), generator=gen).to(t).cuda()
    k, v = states[:, :, 0].transpose(1, 2), states[:, :, 1].transpose(1, 2)
    lengths = torch.tensor([150, 65], dtype=torch.int32, device="cuda")
    table = torch.tensor([[4, 0, 3], [1, 2, -1]], dtype=torch.int32, device="cuda")
    pool = [torch.zeros((5, heads, 64, d), dtype=torch.uint8, device="cuda"),
            torch.zeros((5, heads, d, 64), dtype=torch.uint8, device="cuda"),
            torch.zeros((5, heads), device="cuda"), torch.zeros((5, heads), device="cuda")]
    lc.kv_cache_store(k, v, table, lengths, *pool)
    at = table.clamp_min(0).long()
    kc = (pool[0][at].view(torch.float8_e4m3fn).float() * pool[2][at][..., None, None]).permute(0, 2, 1, 3, 4)
    vc = (pool[1][at].view(torch.float8_e4m3fn).float() * pool[3][at][..., None, None]).transpose(3, 4)
    kc = kc.reshape(b, heads, 192, d)
    vc = vc.permute(0, 2, 1, 3, 4).reshape(b, heads, 192, d)
    q = torch.randn((b, heads, 6, d), generator=gen).to(t).cuda()
    ref = Attention(q, kc, vc, lengths)
    ref.up = 2.0**-16
    for i in range(6):
        out = lc.kv_cache_attention(q[:, :, i:i + 1], *pool, table, lengths)
        bound = (ref.out_bound() + 2.0**-20 * (ref.p @ ref.v.abs()))[:, :, i:i + 1]
        assert_within(out, ref.out[:, :, i:i + 1], bound, f"token {i}")
    whole = lc.kv_cache_attention(q, *pool, table, lengths)
    assert_within(whole, ref.out, ref.out_bound() + 2.0**-20 * (ref.p @ ref.v.abs()), "all tokens")
