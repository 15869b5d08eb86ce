"""Cross attention and its gradients against 64 bits, element by element, within
bounds that follow from the roundings (decoder_ref.py): lengths from none and one
to several tiles, sizes off every tile, heads that share keys, strides and bases
that suit no vector load, padded rows full of NaN, offsets past 32 bits; graphs,
streams and bits that do not change from call to call.
"""
import math

import numpy as np
import pytest
import torch

from decoder_ref import Attention, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _tensor(gen, b, h, s, d, dtype, layout="bhsd", offset=0, pad=0):
    """[b, h, s, d] on the GPU.  pad: unused values behind each row; offset: the
    base lies so many values into its memory."""
    w = d + pad
    shape = (b, s, h, w) if layout == "bshd" else (b, h, s, w)
    n = math.prod(shape)
    mem = torch.full((n + offset,), math.nan, dtype=dtype)
    mem[offset:] = torch.randn(n, generator=gen).to(dtype)
    x = mem.cuda()[offset:].view(shape)
    if layout == "bshd":
        x = x.transpose(1, 2)
    return x[..., :d]


def _check(lc, q, k, v, lengths=None, scale=None, dout=None, seed=0, what=""):
    ref = Attention(q, k, v, lengths, scale)
    print(f"[case] {what} q{tuple(q.shape)} k{tuple(k.shape)} {q.dtype} forward", flush=True)
    out, lse = lc.cross_attention(q, k, v, lengths, scale=scale, return_lse=True)
    torch.cuda.synchronize()
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    assert_within(out, ref.out, ref.out_bound(), f"{what} out")
    assert_within(lse, ref.lse, ref.lse_bound(), f"{what} lse")
    if dout is None:
        dout = torch.randn(q.shape, generator=_gen(seed + 1000)).to(q.dtype).cuda()
    print(f"[case] {what} backward", flush=True)
    got = lc.cross_attention_backward(dout, q, k, v, out, lse, lengths, scale=scale)
    torch.cuda.synchronize()
    for name, x in zip(("dq", "dk", "dv"), got):
        g, bound = ref.backward(dout)[name]
        assert x.dtype == q.dtype
        assert_within(x, g, bound, f"{what} {name}")
    return out, lse, got


SHAPES = [
    # b, hq, hkv, sq, sk, d, lengths
    (1, 1, 1, 1, 1, 64, None),
    (1, 2, 2, 1, 2, 64, None),
    (2, 4, 2, 3, 5, 32, [0, 5]),
    (3, 2, 2, 4, 9, 64, [1, 9, 0]),
    (1, 12, 12, 1, 196, 64, None),      # one token, one image
    (2, 8, 2, 77, 1000, 64, [1000, 501]),
    (1, 4, 1, 130, 63, 128, None),      # rows of a head cross row blocks
    (2, 2, 2, 128, 64, 128, None),      # whole tiles
    (2, 2, 2, 128, 128, 64, [128, 127]),
    (1, 3, 1, 129, 65, 80, None),
    (3, 2, 1, 31, 33, 40, [33, 32, 31]),
    (1, 1, 1, 5, 257, 128, None),
    (1, 8, 1, 1, 700, 128, None),       # one token, eight heads to a key head
    (2, 2, 1, 300, 17, 96, [17, 2]),    # many rows, few keys
    (1, 2, 2, 500, 300, 128, None),
    (8, 8, 8, 140, 140, 64, None),      # no split
    (1, 1, 1, 7, 40, 1, None),
    (1, 2, 1, 65, 66, 33, None),        # rows that no vector load suits
    (2, 2, 1, 40, 90, 127, [90, 3]),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(str(x) for x in s[:6]))
def test_against_64_bits(lc, shape, dtype):
    b, hq, hkv, sq, sk, d, lens = shape
    gen = _gen(sq * 1000 + sk + d)
    t = DTYPES[dtype]
    layout = "bshd" if sq % 2 else "bhsd"
    q = _tensor(gen, b, hq, sq, d, t, layout)
    k = _tensor(gen, b, hkv, sk, d, t, layout)
    v = _tensor(gen, b, hkv, sk, d, t, "bhsd")
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    _check(lc, q, k, v, lengths, what=f"{shape} {dtype}")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [
    (4, 8, 8, 1100, 200, 64, [200, 131, 64, 0]),  # 128-row blocks, keys split
    (4, 8, 8, 1100, 70, 128, [70, 65, 64, 1]),
    (16, 8, 8, 640, 40, 64, None),                # enough of them: no split
    (2, 64, 4, 300, 130, 128, [130, 129]),        # rows of a head cross blocks
    (4, 8, 8, 1100, 66, 33, None),                # rows that no vector load suits
], ids=lambda s: "x".join(str(x) for x in s[:6]))
def test_many_rows_against_64_bits(lc, shape, dtype):
    b, hq, hkv, sq, sk, d, lens = shape
    gen = _gen(sq + sk + d)
    t = DTYPES[dtype]
    q = _tensor(gen, b, hq, sq, d, t, "bshd")
    k, v = (_tensor(gen, b, hkv, sk, d, t, x) for x in ("bhsd", "bshd"))
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    if lens is not None:
        for i, n in enumerate(lens):
            k[i, :, n:] = math.nan
            v[i, :, n:] = math.nan
    _check(lc, q, k, v, lengths, what=f"{shape} {dtype}")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_bases_and_strides_off_alignment(lc, dtype):
    gen = _gen(7)
    t = DTYPES[dtype]
    q = _tensor(gen, 2, 4, 35, 64, t, "bshd", offset=1)
    k = _tensor(gen, 2, 2, 70, 64, t, "bhsd", offset=3, pad=5)
    v = _tensor(gen, 2, 2, 70, 64, t, "bshd", pad=1)
    _check(lc, q, k, v, torch.tensor([70, 41], dtype=torch.int32, device="cuda"), what=f"off alignment {dtype}")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_broadcast_inputs(lc, dtype):
    """Strides of zero: one image's states for every row of a batch, one query
    for every position."""
    gen = _gen(8)
    t = DTYPES[dtype]
    q = _tensor(gen, 3, 2, 1, 64, t).expand(3, 2, 20, 64)
    k = _tensor(gen, 1, 1, 50, 64, t).expand(3, 2, 50, 64)
    v = _tensor(gen, 1, 1, 50, 64, t).expand(3, 2, 50, 64)
    _check(lc, q, k, v, torch.tensor([50, 20, 1], dtype=torch.int32, device="cuda"), what=f"broadcast {dtype}")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d", [64, 37])
def test_padding_may_hold_anything(lc, dtype, d):
    """NaN and infinities in keys and values past a row's length change nothing."""
    gen = _gen(9)
    t = DTYPES[dtype]
    q = _tensor(gen, 3, 2, 33, d, t)
    k = _tensor(gen, 3, 2, 100, d, t)
    v = _tensor(gen, 3, 2, 100, d, t)
    lens = [100, 67, 0]
    for i, n in enumerate(lens):
        k[i, :, n:] = math.nan
        v[i, :, n:] = math.inf
    _check(lc, q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), what=f"padding {dtype}")


def test_lengths_are_held_to_the_tensors(lc):
    gen = _gen(10)
    q, k, v = (_tensor(gen, 3, 1, s, 64, torch.bfloat16) for s in (5, 30, 30))
    wild = torch.tensor([-4, 2**31 - 1, 12], dtype=torch.int32, device="cuda")
    held = torch.tensor([0, 30, 12], dtype=torch.int32, device="cuda")
    a, b = (lc.cross_attention(q, k, v, n, return_lse=True) for n in (wild, held))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    _check(lc, q, k, v, wild, what="wild lengths")


def test_nothing_to_attend_to_and_nothing_to_ask(lc):
    t = torch.float16
    q = torch.randn(2, 4, 3, 64, device="cuda").to(t)
    none = torch.empty(2, 2, 0, 64, device="cuda", dtype=t)
    out, lse = lc.cross_attention(q, none, none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = lc.cross_attention_backward(q, q, none, none, out, lse)
    assert (dq == 0).all() and dk.shape == none.shape and dv.shape == none.shape
    k = torch.randn(2, 2, 9, 64, device="cuda").to(t)
    none = torch.empty(2, 4, 0, 64, device="cuda", dtype=t)
    out, lse = lc.cross_attention(none, k, k, return_lse=True)
    assert out.shape == none.shape and lse.shape == (2, 4, 0)
    dq, dk, dv = lc.cross_attention_backward(none, none, k, k, out, lse)
    assert dq.shape == none.shape and (dk == 0).all() and (dv == 0).all()
    none = torch.empty(0, 4, 3, 64, device="cuda", dtype=t)
    kv = torch.empty(0, 2, 9, 64, device="cuda", dtype=t)
    assert lc.cross_attention(none, kv, kv).shape == none.shape


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("scale", [-0.3, 2.0, 1e-3])
def test_scales(lc, dtype, scale):
    gen = _gen(11)
    t = DTYPES[dtype]
    q, k, v = (_tensor(gen, 1, 2, s, 48, t) for s in (40, 75, 75))
    _check(lc, q, k, v, scale=scale, what=f"scale {scale} {dtype}")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_scores_far_apart(lc, dtype):
    """Rows whose maximum moves by hundreds from tile to tile, up and down, and
    scores far below zero."""
    t = DTYPES[dtype]
    gen = _gen(12)
    q = _tensor(gen, 1, 1, 64, 64, t) * 0.25
    k = _tensor(gen, 1, 1, 400, 64, t) * 0.25
    v = _tensor(gen, 1, 1, 400, 64, t)
    q[..., 0] = 8
    ramp = torch.linspace(-300, 300, 400)
    k[0, 0, :, 0] = torch.cat([ramp[::2], ramp.flip(0)[1::2]]).to(t).cuda()
    _check(lc, q, k, v, what=f"ramp {dtype}")
    k[0, 0, :, 0] = -300
    _check(lc, q, k, v, what=f"far below {dtype}")


@pytest.mark.parametrize("size", [1e-6, 1.0, 2000.0])
@pytest.mark.parametrize("sq,sk", [(64, 700), (300, 64)])
def test_f16_gradients_of_any_size(lc, size, sq, sk):
    """dO far from one: dS would be below fp16's range, or above it."""
    gen = _gen(13)
    q, k, v = (_tensor(gen, 1, 2, s, 64, torch.float16) for s in (sq, sk, sk))
    dout = (torch.randn(q.shape, generator=gen) * size)
    # rows of very different size, and one of zeros
    dout[..., ::3, :] *= 2.0**-6
    dout[..., 1, :] = 0
    _check(lc, q, k, v, dout=dout.to(torch.float16).cuda(), what=f"dout {size}")


def test_gradient_against_differences(lc):
    """fp32 gradients against central differences of the 64-bit forward."""
    gen = _gen(14)
    q, k, v = (_tensor(gen, 1, 2, s, 16, torch.float32) for s in (6, 11, 11))
    lengths = torch.tensor([9], dtype=torch.int32, device="cuda")
    dout = torch.randn(q.shape, generator=gen).cuda()
    out, lse = lc.cross_attention(q, k, v, lengths, return_lse=True)
    grads = lc.cross_attention_backward(dout, q, k, v, out, lse, lengths)

    h = 2.0**-14  # the third derivative's share is h^2, of order 1e-9
    for which, g in enumerate(grads):
        for at in range(0, g.numel(), 29):
            ends = []
            for step in (h, -h):
                x = [t.double().clone() for t in (q, k, v)]
                x[which].view(-1)[at] += step
                ends.append((_plain(*x, lengths) * dout.double()).sum().item())
            want = (ends[0] - ends[1]) / (2 * h)
            # fp32 gradients of terms of order 10 over 11 keys and 16 columns
            assert abs(g.reshape(-1)[at].item() - want) < 2e-5, (which, at)


def _plain(q, k, v, lengths):
    s = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
    hidden = torch.arange(k.shape[2], device=k.device) >= lengths.view(-1, 1, 1, 1)
    return torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v


def test_offsets_past_32_bits(lc):
    """Rows 8 M values apart, the widest that is taken: a head's keys span 9 GB."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    gen = _gen(15)
    stride, sk = 8_000_000, 600
    mem = torch.empty(sk * stride, dtype=torch.bfloat16, device="cuda")
    k = mem.as_strided((1, 1, sk, 64), (0, 0, stride, 1))
    v = mem.as_strided((1, 1, sk, 64), (0, 0, stride, 1), 64)
    k.copy_(torch.randn(k.shape, generator=gen))
    v.copy_(torch.randn(v.shape, generator=gen))
    q = _tensor(gen, 1, 1, 20, 64, torch.bfloat16)
    kc, vc = k.contiguous(), v.contiguous()
    out, lse = lc.cross_attention(q, k, v, return_lse=True)
    near, lse2 = lc.cross_attention(q, kc, vc, return_lse=True)
    assert torch.equal(out, near) and torch.equal(lse, lse2)
    far = lc.cross_attention_backward(q, q, k.expand(1, 1, sk, 64), v, out, lse)
    near = lc.cross_attention_backward(q, q, kc, vc, out, lse)
    assert all(torch.equal(x, y) for x, y in zip(far, near))


def test_a_capture_may_be_the_first_call():
    """In a process of its own: the library's first call of all is captured."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys
sys.path.insert(0, %r)
import torch
q, k = (torch.randn(1, 2, s, 64, device="cuda") for s in (5, 700))
x = torch.randn(9, 64, device="cuda")
torch.cuda.synchronize()
import lightning_core as lc
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = lc.cross_attention(q, k, k)
    y = lc.layer_norm(x)
for _ in range(3):
    q.normal_(); x.normal_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, lc.cross_attention(q, k, k)) and torch.equal(y, lc.layer_norm(x))
print("fine")
""" % os.path.join(root, "lightining-core_amd")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout[-500:] + r.stderr[-1500:]


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_equal_calls_give_equal_bits(lc, dtype):
    gen = _gen(16)
    t = DTYPES[dtype]
    q, k, v = (_tensor(gen, 2, h, s, 64, t) for h, s in ((4, 70), (2, 900), (2, 900)))
    first = None
    for _ in range(3):
        out, lse = lc.cross_attention(q, k, v, return_lse=True)
        got = (out, lse) + tuple(lc.cross_attention_backward(out, q, k, v, out, lse))
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))


def test_captured_graphs_replay(lc):
    """Two graphs with workspaces of their own, replayed with eager work between,
    on inputs that change."""
    gen = _gen(17)
    sets = [[_tensor(gen, 1, 4, s, 64, torch.bfloat16) for s in (9, 800, 800, 9)] for _ in range(2)]
    graphs, results = [], []
    for q, k, v, g in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = lc.cross_attention(q, k, v, return_lse=True)
            grads = lc.cross_attention_backward(g, q, k, v, out, lse)
        graphs.append(graph)
        results.append((out, lse) + tuple(grads))
    for turn in range(4):
        for x in sets[0] + sets[1]:
            x.copy_(torch.randn(x.shape, generator=gen))
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        for (q, k, v, g), got in zip(sets, results):
            out, lse = lc.cross_attention(q, k, v, return_lse=True)
            want = (out, lse) + tuple(lc.cross_attention_backward(g, q, k, v, out, lse))
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), turn


def test_runs_on_the_current_stream(lc):
    gen = _gen(18)
    q, k, v = (_tensor(gen, 2, 4, s, 64, torch.float16) for s in (50, 600, 600))
    want = lc.cross_attention(q, k, v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            # filled behind a long copy of the same stream: an earlier launch would read zeros
            x = torch.zeros_like(q)
            torch.empty(256 << 20, dtype=torch.uint8, device="cuda").fill_(1)
            x.copy_(q)
            results.append((x, lc.cross_attention(x, k, v)))
    torch.cuda.synchronize()
    for _, got in results:
        assert torch.equal(got, want)


def test_output_tensor_of_the_caller(lc):
    gen = _gen(19)
    q, k, v = (_tensor(gen, 2, 4, s, 64, torch.bfloat16) for s in (5, 60, 60))
    want = lc.cross_attention(q, k, v)
    big = torch.full((2, 5, 4, 70), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big.transpose(1, 2)[..., :64]
    assert lc.cross_attention(q, k, v, out=out) is out
    assert torch.equal(out, want) and (big[..., 64:] == 7).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_numpy_arrays(lc, dtype):
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal((2, h, s, 40)).astype(dtype) for h, s in ((4, 9), (2, 30), (2, 30)))
    lens = np.array([30, 11])
    out, lse = lc.cross_attention(q, k, v, lens, return_lse=True)
    assert isinstance(out, np.ndarray) and out.dtype == dtype
    grads = lc.cross_attention_backward(out, q, k, v, out, lse, lens)
    tq, tk, tv = (torch.from_numpy(x).cuda() for x in (q, k, v))
    tl = torch.from_numpy(lens.astype(np.int32)).cuda()
    tout, tlse = lc.cross_attention(tq, tk, tv, tl, return_lse=True)
    want = lc.cross_attention_backward(tout, tq, tk, tv, tout, tlse, tl)
    for x, y in zip((out, lse) + tuple(grads), (tout, tlse) + tuple(want)):
        assert np.array_equal(x, y.cpu().numpy())


def test_refusals_on_the_gpu(lc):
    q, k, v = (torch.randn(1, 2, s, 64, device="cuda") for s in (3, 9, 9))
    with pytest.raises(ValueError, match="cpu"):
        lc.cross_attention(q, k.cpu(), v)
    with pytest.raises(ValueError, match="int32"):
        lc.cross_attention(q, k, v, torch.tensor([3], device="cuda"))
    with pytest.raises(ValueError, match="one type"):
        lc.cross_attention(q, k, v.half())
    with pytest.raises(ValueError, match="contiguous"):
        lc.cross_attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v)
    with pytest.raises(RuntimeError, match="overlapping"):
        lc.cross_attention(q, k, v, out=torch.empty(1, 2, 1, 64, device="cuda").expand(1, 2, 3, 64))
    # a host pointer at the C interface is an error, not a fault
    import ctypes

    from lightning_core import _native as N
    host = np.zeros((1, 2, 3, 64), np.float32)
    cfg = N.CrossAttentionConfig(1, 2, 2, 3, 9, 64, N.LC_DTYPE_F32, 0.0)

    def t(p, s):
        return ctypes.byref(N.DeviceTensor(p, 2 * s * 64, s * 64, 64))
    ok = (t(q.data_ptr(), 3), t(k.data_ptr(), 9), t(v.data_ptr(), 9))
    out = t(host.ctypes.data, 3)
    lib = N.load()
    assert lib.lcCrossAttentionForward(ctypes.byref(cfg), *ok, None, out, None, None, 0, None) == N.LC_INVALID_VALUE
    assert b"out is not memory of device" in lib.lcGetLastErrorMessage()
    big = N.CrossAttentionConfig(1, 2, 2, 3, 900, 64, N.LC_DTYPE_F32, 0.0)
    long = (t(q.data_ptr(), 3), t(k.data_ptr(), 0), t(v.data_ptr(), 0))
    good = torch.empty_like(q)
    assert lib.lcCrossAttentionForward(ctypes.byref(big), *long, None, t(good.data_ptr(), 3), None, None, 0,
                                       None) == N.LC_INVALID_VALUE
    assert b"workspace needs" in lib.lcGetLastErrorMessage()
