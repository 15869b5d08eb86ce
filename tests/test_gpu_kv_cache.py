"""The 8-bit paged cache: what a store writes, code by code, and attention over
it against 64 bits on the values that the codes stand for.

Codes: an e4m3 code is the nearest to x / scale with fp32 scale and quotient, so
it is off by half a step (2^-4 of the value; 2^-10 below the normal numbers) and
the quotient's two roundings.
"""
import math

import numpy as np
import pytest
import torch

from decoder_ref import Attention, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAGE = 64


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _pool(pages, heads, d, fill=0x55):
    return [torch.full((pages, heads, PAGE, d), fill, dtype=torch.uint8, device="cuda"),
            torch.full((pages, heads, d, PAGE), fill, dtype=torch.uint8, device="cuda"),
            torch.full((pages, heads), 9.0, device="cuda"), torch.full((pages, heads), 9.0, device="cuda")]


def _table(lengths, spare, gen, width=None):
    need = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max([width or 1] + need)), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def _values(pool, table, lengths):
    """The cache's keys and values for each row, 64 bits, [b, h, width * 64, d]."""
    out = []
    for codes, scales, transposed in ((pool[0], pool[2], False), (pool[1], pool[3], True)):
        pages, h = codes.shape[:2]
        d = codes.shape[2] if transposed else codes.shape[3]
        x = torch.zeros((table.shape[0], h, table.shape[1] * PAGE, d), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            for p in range(-(-n // PAGE)):
                at = int(table[b, p])
                page = codes[at].view(torch.float8_e4m3fn).double() * scales[at].double().view(-1, 1, 1)
                m = min(PAGE, n - p * PAGE)
                page = page.transpose(1, 2) if transposed else page
                x[b, :, p * PAGE:p * PAGE + m] = page[:, :m]
        out.append(x)
    return out


STORES = [
    # heads, d, lengths, padded length
    (1, 16, [1], 1),
    (2, 64, [64, 63], 64),
    (3, 48, [130, 0, 65], 130),
    (12, 64, [196, 196], 196),
    (2, 128, [500, 257, 1], 500),
    (1, 80, [64, 128], 200),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layout", ["bhsd", "bshd", "odd"])
@pytest.mark.parametrize("case", STORES, ids=str)
def test_store(lc, case, layout, dtype):
    h, d, lengths, sk = case
    gen = _gen(d + sk)
    b = len(lengths)
    table, pages = _table(lengths, 2, gen, -(-sk // PAGE))
    tables = table.cuda()

    def make():
        if layout == "bshd":
            x = torch.randn((b, sk, h, d), generator=gen).to(DTYPES[dtype]).cuda().transpose(1, 2)
        elif layout == "odd":  # rows that no vector load suits
            x = torch.randn((b, h, sk, d + 1), generator=gen).to(DTYPES[dtype]).cuda()[..., 1:]
        else:
            x = torch.randn((b, h, sk, d), generator=gen).to(DTYPES[dtype]).cuda()
        return x

    k, v = make() * 3, make()
    for i, n in enumerate(lengths):  # what lies past a length is not read into anything
        k[i, :, n:] = math.nan
        v[i, :, n:] = math.inf
    pool = _pool(pages, h, d)
    kv = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    print(f"[case] store {case} {layout} {dtype}", flush=True)
    lc.kv_cache_store(k, v, tables, kv, *pool)
    torch.cuda.synchronize()
    used = set()
    for i, n in enumerate(lengths):
        for p in range(-(-n // PAGE)):
            at, m = int(table[i, p]), min(PAGE, n - p * PAGE)
            used.add(at)
            for x, codes, scales, transposed in ((k, pool[0], pool[2], False), (v, pool[1], pool[3], True)):
                rows = x[i, :, p * PAGE:p * PAGE + m].double()
                scale = (rows.abs().amax((1, 2)) / 448).clamp_min(2.0**-126)
                assert_within(scales[at], scale, scale * 2.0**-23, "scale")
                got = codes[at].transpose(1, 2) if transposed else codes[at]
                assert (got[:, m:].view(torch.uint8) & 0x7F == 0).all()  # the rest of a last page
                got = got[:, :m].contiguous().view(torch.float8_e4m3fn).double()
                want = rows / scale.view(-1, 1, 1)
                assert_within(got, want, want.abs() * (2.0**-4 + 2.0**-22) + 2.0**-10, "codes")
    for at in set(range(pages)) - used:  # pages that no row names
        assert (pool[0][at] == 0x55).all() and (pool[1][at] == 0x55).all()
        assert (pool[2][at] == 9).all() and (pool[3][at] == 9).all()


def test_codes_are_the_nearest(lc):
    """Values on and next to every border between codes, ties to even: the codes
    of torch's own conversion of the quotient."""
    x = torch.arange(0, 449, 1.0)
    steps = torch.cat([x, x + 0.5, x / 64, x / 512, x / 4096, torch.tensor([2.0**-10, 3 * 2.0**-10, 2.0**-11])])
    steps = torch.cat([steps, steps * (1 + 2.0**-20), steps * (1 - 2.0**-20)]).clamp(max=448.0)
    rows = -(-len(steps) // 64) * 64
    flat = torch.zeros(rows, dtype=torch.float32)
    flat[:len(steps)] = steps
    flat = flat.view(-1, 16)  # [tokens, d]
    tokens = flat.shape[0]
    pages = -(-tokens // PAGE)
    k = flat.view(1, 1, tokens, 16).clone()
    k[0, 0, ::PAGE, 0] = 448.0  # every page's scale is one
    k[0, 0, 1::2] *= -1
    k = k.cuda()
    pool = _pool(pages, 1, 16)
    lc.kv_cache_store(k, k, torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1), None, *pool)
    want = k[0, 0].to(torch.float8_e4m3fn).view(torch.uint8)
    assert (pool[2] == 1).all()
    assert torch.equal(pool[0].view(-1, 16)[:tokens], want)
    assert torch.equal(pool[1].transpose(2, 3).reshape(-1, 16)[:tokens], want)


def test_pages_of_zeros_and_of_tiny_values(lc):
    k = torch.zeros(1, 1, 128, 32, device="cuda")
    k[0, 0, 64:] = torch.randn(64, 32, generator=_gen(3)).cuda() * 1e-41
    pool = _pool(2, 1, 32)
    lc.kv_cache_store(k, k, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), None, *pool)
    assert (pool[0][0] & 0x7F == 0).all() and (pool[2][:, 0] == 2.0**-126).all()
    out = lc.kv_cache_attention(torch.ones(1, 1, 1, 32, device="cuda"), *pool,
                                torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"))
    assert torch.isfinite(out).all()


ATTENTIONS = [
    # hq, hkv, sq, d, lengths, width of the table (0: as needed)
    (1, 1, 1, 16, [1], 0),
    (12, 12, 1, 64, [196] * 3, 0),
    (4, 2, 1, 64, [0, 64, 65, 1], 0),
    (8, 1, 2, 128, [1000, 129], 0),
    (8, 8, 3, 48, [63, 300], 9),
    (16, 2, 5, 80, [130, 7], 0),      # rows of a head block cross 16
    (2, 2, 40, 112, [90], 0),
    (16, 2, 5, 64, [200, 7], 0),      # blocks of rows that share whole pages' width
    (8, 1, 3, 128, [130, 64, 0], 0),
    (32, 4, 1, 128, [4000, 1], 0),    # splits, and rows without their share
    (1, 1, 1, 32, [6400], 200),
    (2, 1, 1, 64, list(range(131)), 0),   # every length of a last page
    (3, 1, 6, 128, list(range(131)), 0),
    (2, 1, 1, 80, list(range(131)), 0),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", ATTENTIONS, ids=lambda c: str(c)[:40])
def test_attention(lc, case, dtype):
    hq, hkv, sq, d, lengths, width = case
    gen = _gen(hq + d + sum(lengths))
    b = len(lengths)
    table, pages = _table(lengths, 1, gen, width)
    pool = _pool(pages, hkv, d, 0x7F)  # NaN codes wherever nothing was stored
    pool[0].copy_((torch.randn(pool[0].shape, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
                  .view(torch.uint8))
    pool[1].copy_((torch.randn(pool[1].shape, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
                  .view(torch.uint8))
    pool[2].copy_((torch.rand(pool[2].shape, generator=gen) + 0.5) / 100)
    pool[3].copy_((torch.rand(pool[3].shape, generator=gen) + 0.5) / 100 * 10.0 ** torch.randint(
        -3, 3, pool[3].shape, generator=gen))
    for i, n in enumerate(lengths):  # behind the last token of a last page: NaN
        if n % PAGE:
            at = int(table[i, n // PAGE])
            pool[0][at, :, n % PAGE:] = 0x7F
            pool[1][at, :, :, n % PAGE:] = 0xFF
    q = torch.randn((b, sq, hq, d), generator=gen).to(DTYPES[dtype]).cuda().transpose(1, 2)
    kv = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    print(f"[case] cached {case} {dtype}", flush=True)
    out, lse = lc.kv_cache_attention(q, *pool, table.cuda(), kv, return_lse=True)
    torch.cuda.synchronize()
    k, v = _values(pool, table, lengths)
    # Two bf16 terms of P leave 2^-16 of it, three for fp32 queries (2^-24).
    ref = Attention(q, k, v, kv)
    ref.up = 2.0**-16 if dtype != "f32" else 2.0**-24
    assert out.dtype == q.dtype
    # a key's or value's scale is one more fp32 factor; splitting q and p in terms
    # leaves at most 2^-23 of each
    extra = 2.0**-21 * (ref.p @ ref.v.abs()) + 1e-30
    assert_within(out, ref.out, ref.out_bound() + extra, "out")
    assert_within(lse, ref.lse, ref.lse_bound() + 2.0**-20, "lse")


def test_store_then_attend(lc):
    """A run as a server makes it: store, attend, and the same pages named by
    another row (a fork of the sequence)."""
    gen = _gen(5)
    k, v = (torch.randn((2, 300, 4, 64), generator=gen).bfloat16().cuda().transpose(1, 2) for _ in range(2))
    lengths = [300, 70]
    table, pages = _table(lengths, 0, gen)
    pool = _pool(pages, 4, 64)
    kv = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    lc.kv_cache_store(k, v, table.cuda(), kv, *pool)
    table3 = torch.cat([table, table[:1]]).cuda()
    kv3 = torch.tensor([300, 70, 150], dtype=torch.int32, device="cuda")
    q = torch.randn((3, 8, 1, 64), generator=gen).bfloat16().cuda()
    q[2] = q[0]
    out = lc.kv_cache_attention(q, *pool, table3, kv3)
    whole = lc.cross_attention(q[:2], k, v, kv)
    # e4m3 keeps 2^-4 of a value: scores of unit size move by about that, and the
    # values by as much, averaged over the keys
    assert (out[:2].float() - whole.float()).norm() < 2.0**-3 * whole.float().norm()
    keys, values = _values(pool, table3.cpu(), [300, 70, 150])
    ref = Attention(q, keys, values, kv3)
    assert_within(out, ref.out, ref.out_bound() + 2.0**-14 * (ref.p @ ref.v.abs()), "out")


def test_pages_outside_the_pool(lc):
    gen = _gen(6)
    k = torch.randn((3, 1, 128, 32), generator=gen).cuda()
    pool = _pool(4, 1, 32)
    before = [x.clone() for x in pool]
    table = torch.tensor([[0, 4], [-1, 1], [2, 3]], dtype=torch.int32, device="cuda")
    lc.kv_cache_store(k, k, table, None, *pool)
    torch.cuda.synchronize()
    good = _pool(4, 1, 32)
    lc.kv_cache_store(k[2:], k[2:], table[2:].contiguous(), None, *good)
    for x, y, z in zip(pool, before, good):
        assert not torch.equal(x[0], y[0]) and not torch.equal(x[1], y[1])
        assert torch.equal(x[2:], z[2:])
    q = torch.randn((3, 2, 1, 32), generator=gen).cuda()
    out, lse = lc.kv_cache_attention(q, *pool, table, return_lse=True)
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2]).all()
    # an entry past the length is not used
    kv = torch.tensor([64, 0, 128], dtype=torch.int32, device="cuda")
    out = lc.kv_cache_attention(q, *pool, table, kv)
    assert torch.isfinite(out).all() and (out[1] == 0).all()
    wild = torch.tensor([-5, 0, 2**31 - 1], dtype=torch.int32, device="cuda")
    held = torch.tensor([0, 0, 128], dtype=torch.int32, device="cuda")
    a, b = (lc.kv_cache_attention(q, *pool, table, n) for n in (wild, held))
    assert torch.equal(a, b)


def test_a_pool_past_32_bits(lc):
    """Pages whose bytes lie behind 4 GB."""
    pages, h, d = 70_000, 8, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free memory")
    kp = torch.empty((pages, h, PAGE, d), dtype=torch.uint8, device="cuda")
    vp = torch.empty((pages, h, d, PAGE), dtype=torch.uint8, device="cuda")
    ks, vs = torch.empty((pages, h), device="cuda"), torch.empty((pages, h), device="cuda")
    k, v = (torch.randn((1, h, 100, d), generator=_gen(s)).half().cuda() for s in (1, 2))
    q = torch.randn((1, h, 1, d), generator=_gen(3)).half().cuda()
    far = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    kv = torch.tensor([100], dtype=torch.int32, device="cuda")
    got = []
    for t in (far, near):
        lc.kv_cache_store(k, v, t, kv, kp, vp, ks, vs)
        got.append(lc.kv_cache_attention(q, kp, vp, ks, vs, t, kv))
    assert torch.equal(got[0], got[1])
    assert torch.equal(kp[pages - 1], kp[0]) and torch.equal(vp[pages - 2], vp[1])


def test_equal_bits_graphs_and_streams(lc):
    gen = _gen(9)
    lengths = [2000, 900]
    table, pages = _table(lengths, 0, gen)
    pool = _pool(pages, 2, 64)
    k, v = (torch.randn((2, 2, 2000, 64), generator=gen).half().cuda() for _ in range(2))
    table = table.cuda()
    kv = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn((2, 8, 1, 64), generator=gen).half().cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lc.kv_cache_store(k, v, table, kv, *pool)
        out = lc.kv_cache_attention(q, *pool, table, kv)
    side = torch.cuda.Stream()
    for turn in range(4):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=gen))
        kv.copy_(torch.tensor([2000 - 300 * turn, 900 + turn]))
        graph.replay()
        other = _pool(pages, 2, 64)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lc.kv_cache_store(k, v, table, kv, *other)
            want = lc.kv_cache_attention(q, *other, table, kv)
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn


def test_float8_tensors_and_numpy(lc):
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((1, 2, 100, 32)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, 4, 1, 32)).astype(np.float32)
    table = np.array([[1, 0]])
    pool = [np.zeros((2, 2, PAGE, 32), np.uint8), np.zeros((2, 2, 32, PAGE), np.uint8),
            np.zeros((2, 2), np.float32), np.zeros((2, 2), np.float32)]
    lc.kv_cache_store(k, v, table, [100], *pool)
    out = lc.kv_cache_attention(q, *pool, table, [100])
    tk, tv, tq = (torch.from_numpy(x).cuda() for x in (k, v, q))
    tt = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    kv = torch.tensor([100], dtype=torch.int32, device="cuda")
    tp = _pool(2, 2, 32, 0)
    tp = [tp[0].view(torch.float8_e4m3fn), tp[1].view(torch.float8_e4m3fn), tp[2], tp[3]]
    lc.kv_cache_store(tk, tv, tt, kv, *tp)
    assert np.array_equal(pool[0], tp[0].view(torch.uint8).cpu().numpy())
    assert np.array_equal(pool[3], tp[3].cpu().numpy())
    assert np.array_equal(out, lc.kv_cache_attention(tq, *tp, tt, kv).cpu().numpy())


def test_refusals_on_the_gpu(lc):
    pool = _pool(2, 2, 32)
    k = torch.randn(1, 2, 100, 32, device="cuda")
    t = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="2 needed"):
        lc.kv_cache_store(k, k, t[:, :1].contiguous(), None, *pool)
    with pytest.raises(ValueError, match="agree"):
        lc.kv_cache_store(k[..., :16], k[..., :16], t, None, *pool)
    with pytest.raises(ValueError, match="int32"):
        lc.kv_cache_store(k, k, t.long(), None, *pool)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        lc.kv_cache_store(k[..., :24].contiguous(), k[..., :24].contiguous(), t, None, *_pool(2, 2, 24))
    with pytest.raises(RuntimeError, match="without pages"):
        lc.kv_cache_attention(k[:, :, :1].contiguous(), *_pool(0, 2, 32), t)
    with pytest.raises(ValueError, match="multiple"):
        lc.kv_cache_attention(torch.randn(1, 3, 1, 32, device="cuda"), *pool, t)
