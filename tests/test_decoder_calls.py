"""The compiled call helper of the decoder operators: what reaches an entry point,
and that its route and ctypes' give the same results and the same refusals."""
import ctypes

import pytest
import torch

import lightning_core as lc
from lightning_core import _decoder

invoke = _decoder._invoke
needs_helper = pytest.mark.skipif(invoke is None, reason="the compiled helper is not built")


class _View(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("sb", ctypes.c_int64), ("sh", ctypes.c_int64), ("ss", ctypes.c_int64)]


@pytest.fixture
def entry():
    seen = []

    def call(*args):
        seen.append([ctypes.c_int64(a).value for a in args])
        tensors = seen[-1][0]
        if 0 < tensors <= 3:  # the first argument says how many structures follow it
            seen[-1].append([(v.data or 0, v.sb, v.sh, v.ss) for v in
                             (_View.from_address(a) for a in args[1:1 + tensors])])
        return 7
    proto = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_int64] * 16)
    fn = proto(call)
    yield ctypes.cast(fn, ctypes.c_void_p).value, seen
    del fn


@needs_helper
def test_arguments_reach_the_entry_point(entry):
    at, seen = entry
    x = torch.zeros(2, 5, 3, 8)
    y = x.transpose(1, 2)
    one = torch.zeros(2, 3, 4, 2)[..., :1]  # one value a row, at a stride of 2 rows' values
    assert invoke(at, "itttpp", 3, x, y, one, None, x) == 7
    got = seen[0]
    assert got[0] == 3 and got[4] == 0 and got[5] == x.data_ptr() and got[6:16] == [0] * 10
    assert got[16] == [(t.data_ptr(), *t.stride()[:3]) for t in (x, y, one)]


@needs_helper
@pytest.mark.parametrize("value", [0, 1, -1, 2 ** 31, 2 ** 40 + 1, -2 ** 63, 2 ** 63 + 5, 2 ** 64 - 1])
def test_integers_travel_whole(entry, value):
    at, seen = entry
    assert invoke(at, "ii", 0, value) == 7
    assert seen[0][1] == ctypes.c_int64(value).value


@needs_helper
def test_refusals_before_the_call(entry):
    at, seen = entry
    x = torch.zeros(2, 3, 4, 8)
    assert invoke(at, "itt", 0, x, x.transpose(2, 3)) == -2
    assert invoke(at, "itt", 0, x.transpose(2, 3), x) == -1
    assert invoke(at, "it", 0, x[..., :1].transpose(2, 3)) == -1 - 0  # rows of 4 values, 8 apart
    with pytest.raises(ValueError):
        invoke(at, "it", 0, x[0])
    with pytest.raises(AttributeError):
        invoke(at, "ip", 0, 5)
    with pytest.raises(TypeError):
        invoke(at, "ii", 0, None)
    with pytest.raises(TypeError):
        invoke(at, "ii", 0)
    with pytest.raises(TypeError):
        invoke(at, "i" * 17, *range(17))
    with pytest.raises((TypeError, OverflowError)):
        invoke(at, "ii", 0, 2 ** 64)
    with pytest.raises(TypeError):
        invoke(at)
    assert not seen


def _calls():
    g = torch.Generator().manual_seed(11)

    def r(*shape):
        return torch.randn(*shape, generator=g).to("cuda", torch.bfloat16)
    q, k, v, do = r(2, 4, 5, 64), r(2, 2, 70, 64), r(2, 2, 70, 64), r(2, 4, 5, 64)
    n = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    w, x, dy = r(96), r(7, 96), r(7, 96)
    out, lse = lc.cross_attention(q, k, v, n, return_lse=True)
    got = [out, lse, *lc.cross_attention_backward(do, q, k, v, out, lse, n)]
    y, mean, rstd = lc.layer_norm(x, w, w, return_stats=True)
    got += [y, mean, rstd, *lc.layer_norm_backward(dy, x, w, mean, rstd)]
    table = torch.tensor([[1, 0], [2, 3]], dtype=torch.int32, device="cuda")
    pool = [torch.zeros(4, 2, 64, 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
    pool += [torch.zeros(4, 2, device="cuda") for _ in range(2)]
    lc.kv_cache_store(k, v, table, n, *pool)
    got += pool + list(lc.kv_cache_attention(q, *pool, table, n, return_lse=True))
    return got


@needs_helper
@pytest.mark.gpu
def test_both_routes_give_the_same_bits(monkeypatch):
    a = _calls()
    monkeypatch.setattr(_decoder, "_invoke", None)
    b = _calls()
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), i


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_both_routes_refuse_alike(monkeypatch, compiled):
    if not compiled:
        monkeypatch.setattr(_decoder, "_invoke", None)
    q = torch.zeros(1, 2, 3, 64, device="cuda")
    bad = torch.zeros(1, 2, 64, 3, device="cuda").transpose(2, 3)
    for args, name in (((bad, q, q), "q"), ((q, bad, q), "k"), ((q, q, bad), "v")):
        with pytest.raises(ValueError, match=f"^{name}'s last dimension must be contiguous"):
            lc.cross_attention(*args)
    with pytest.raises(ValueError, match="^out's last dimension"):
        lc.cross_attention(q, q, q, out=bad)
    wide = torch.zeros(1, 2, 3, 1000, device="cuda")  # a head size that the library refuses
    with pytest.raises(RuntimeError):
        lc.cross_attention(wide, wide, wide)


@pytest.mark.gpu
def test_threads_on_streams_of_their_own():
    """Two threads call at once, each on its own stream; the results are the bits of one alone."""
    import threading
    want = _calls()
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got[i].append(_calls())
                stream.synchronize()
        except Exception as e:  # shown by the assertion below
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for results in got:
        assert len(results) == 10
        for r in results:
            assert all(torch.equal(x, y) for x, y in zip(r, want))
