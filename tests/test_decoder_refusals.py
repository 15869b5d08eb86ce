"""What the decoder operators refuse before any device work (CPU only): shapes,
types, layouts and sizes at the Python surface, and at the C interface the checks
that come before the device is touched.
"""
import ctypes

import numpy as np
import pytest

import lightning_core as lc
from lightning_core import _native as N


def _cfg(b=1, h=2, hkv=1, sq=3, sk=9, d=64, t=N.LC_DTYPE_F16, scale=0.0):
    return N.CrossAttentionConfig(b, h, hkv, sq, sk, d, t, scale)


def _size(cfg, backward=0):
    n = ctypes.c_size_t(77)
    st = N.load().lcCrossAttentionWorkspaceSize(ctypes.byref(cfg), backward, ctypes.byref(n))
    return st, n.value


@pytest.mark.parametrize("change,status", [
    (dict(h=0), N.LC_INVALID_VALUE), (dict(hkv=0), N.LC_INVALID_VALUE), (dict(d=0), N.LC_INVALID_VALUE),
    (dict(h=3, hkv=2), N.LC_INVALID_VALUE), (dict(t=3), N.LC_INVALID_VALUE),
    (dict(scale=float("nan")), N.LC_INVALID_VALUE), (dict(scale=float("inf")), N.LC_INVALID_VALUE),
    (dict(d=129), N.LC_NOT_SUPPORTED), (dict(sq=1 << 40), N.LC_NOT_SUPPORTED), (dict(sk=1 << 31), N.LC_NOT_SUPPORTED),
    (dict(b=1 << 40), N.LC_NOT_SUPPORTED),
])
def test_cross_attention_configurations(change, status):
    assert _size(_cfg(**change)) == (status, 0)


def test_cross_attention_workspace():
    # few row blocks: the keys are split, and each split keeps a row and two statistics
    st, n = _size(_cfg(b=1, h=12, hkv=12, sq=1, sk=30000))
    assert st == 0 and n > 0 and n % (12 * (64 + 2) * 4) == 0
    assert _size(_cfg(b=64, h=16, hkv=16, sq=200, sk=4096)) == (0, 0)  # enough of them
    st, n = _size(_cfg(b=64, h=16, hkv=16, sq=200, sk=4096), 1)
    assert st == 0 and n == 64 * 16 * 200 * 2 * 4                      # each row's delta
    assert _size(_cfg(sq=0)) == (0, 0) and _size(_cfg(sk=0)) == (0, 0) and _size(_cfg(b=0)) == (0, 0)
    assert N.load().lcCrossAttentionWorkspaceSize(None, 0, ctypes.byref(ctypes.c_size_t())) == N.LC_INVALID_VALUE
    assert N.load().lcCrossAttentionWorkspaceSize(ctypes.byref(_cfg()), 0, None) == N.LC_INVALID_VALUE


def test_cross_attention_tensors():
    """Each is found before the device is opened."""
    lib = N.load()
    cfg = _cfg(sq=2, sk=4)

    def call(q=None, k=None, out=None, cfg=cfg):
        good = dict(q=(256, 256, 128, 64), k=(256, 256, 256, 64), out=(256, 256, 128, 64))
        t = {n: N.DeviceTensor(*(x or good[n])) for n, x in (("q", q), ("k", k), ("out", out))}
        r = ctypes.byref
        st = lib.lcCrossAttentionForward(r(cfg), r(t["q"]), r(t["k"]), r(t["k"]), None, r(t["out"]), None, None, 0, None)
        return st, lib.lcGetLastErrorMessage().decode()

    assert call(q=(None, 256, 128, 64)) == (N.LC_INVALID_VALUE, "cross attention: q has values and a null base")
    assert call(q=(257, 256, 128, 64)) == (N.LC_INVALID_VALUE, "cross attention: q is not aligned to its elements")
    assert call(k=(256, 256, 256, -64)) == (N.LC_INVALID_VALUE, "cross attention: k has a negative stride")
    assert call(out=(256, 256, 128, 63))[0] == N.LC_INVALID_VALUE
    assert call(out=(256, 256, 0, 64))[0] == N.LC_INVALID_VALUE  # two heads written to one place
    assert call(k=(256, 256, 256, 1 << 23))[0] == N.LC_NOT_SUPPORTED  # 128 rows pass 2^31 bytes
    assert lib.lcCrossAttentionForward(ctypes.byref(cfg), None, None, None, None, None, None, None, 0,
                                       None) == N.LC_INVALID_VALUE
    assert lib.lcCrossAttentionBackward(ctypes.byref(cfg), *[None] * 5, None, None, None, None, None, None, 0,
                                        None) == N.LC_INVALID_VALUE


@pytest.mark.parametrize("change,status", [
    (dict(n=0), N.LC_INVALID_VALUE), (dict(t=9), N.LC_INVALID_VALUE), (dict(t=N.LC_DTYPE_F32, w=N.LC_DTYPE_F16),
                                                                        N.LC_INVALID_VALUE),
    (dict(t=N.LC_DTYPE_BF16, w=N.LC_DTYPE_F16), N.LC_INVALID_VALUE), (dict(eps=-1.0), N.LC_INVALID_VALUE),
    (dict(eps=float("nan")), N.LC_INVALID_VALUE), (dict(n=1 << 40), N.LC_NOT_SUPPORTED),
    (dict(rows=1 << 41), N.LC_NOT_SUPPORTED),
])
def test_layer_norm_configurations(change, status):
    a = dict(rows=4, n=32, t=N.LC_DTYPE_F16, w=N.LC_DTYPE_F16, eps=1e-5)
    a.update(change)
    n = ctypes.c_size_t(5)
    cfg = N.LayerNormConfig(a["rows"], a["n"], a["t"], a["w"], a["eps"])
    assert N.load().lcLayerNormWorkspaceSize(ctypes.byref(cfg), ctypes.byref(n)) == status and n.value == 0


def test_layer_norm_tensors():
    lib = N.load()
    cfg = N.LayerNormConfig(4, 32, N.LC_DTYPE_F16, N.LC_DTYPE_F16, 1e-5)
    r = ctypes.byref(cfg)
    inv = N.LC_INVALID_VALUE
    assert lib.lcLayerNormForward(r, None, 32, None, None, 256, 32, None, None, None) == inv
    assert lib.lcLayerNormForward(r, 256, 32, None, None, None, 32, None, None, None) == inv
    assert lib.lcLayerNormForward(r, 256, -32, None, None, 256, 32, None, None, None) == inv
    assert lib.lcLayerNormForward(r, 256, 32, None, None, 256, 31, None, None, None) == inv
    assert lib.lcLayerNormForward(r, 256, 32, 257, None, 256, 32, None, None, None) == inv
    assert lib.lcLayerNormForward(r, 256, 32, None, None, 256, 32, 256, None, None) == inv
    assert lib.lcLayerNormBackward(r, 256, 32, 256, 32, None, None, None, 256, 32, None, None, None, 0, None) == inv


def _pool(**kw):
    a = dict(k=256, v=256, ks=256, vs=256, pages=4, heads=2, d=64)
    a.update(kw)
    return N.KvCache(a["k"], a["v"], a["ks"], a["vs"], a["pages"], a["heads"], a["d"])


@pytest.mark.parametrize("change,status", [
    (dict(heads=0), N.LC_INVALID_VALUE), (dict(d=0), N.LC_INVALID_VALUE), (dict(d=24), N.LC_NOT_SUPPORTED),
    (dict(d=144), N.LC_NOT_SUPPORTED), (dict(k=None), N.LC_INVALID_VALUE), (dict(v=264), N.LC_INVALID_VALUE),
    (dict(ks=258), N.LC_INVALID_VALUE), (dict(pages=1 << 33), N.LC_NOT_SUPPORTED),
])
def test_kv_pools(change, status):
    n = ctypes.c_size_t(5)
    cfg = N.KvAttentionConfig(1, 4, 1, 3, N.LC_DTYPE_F16, 0.0)
    pool = _pool(**change)
    assert N.load().lcKvCacheAttentionWorkspaceSize(ctypes.byref(pool), ctypes.byref(cfg),
                                                    ctypes.byref(n)) == status and n.value == 0


def test_kv_configurations_and_tables():
    lib = N.load()
    pool = _pool()

    def size(*a):
        n = ctypes.c_size_t(5)
        cfg = N.KvAttentionConfig(*a)
        return lib.lcKvCacheAttentionWorkspaceSize(ctypes.byref(pool), ctypes.byref(cfg), ctypes.byref(n)), n.value

    assert size(1, 3, 1, 3, N.LC_DTYPE_F16, 0.0) == (N.LC_INVALID_VALUE, 0)
    assert size(1, 4, 1, 3, 7, 0.0) == (N.LC_INVALID_VALUE, 0)
    assert size(1, 4, 1, 3, N.LC_DTYPE_F16, float("inf")) == (N.LC_INVALID_VALUE, 0)
    assert size(1, 4, 1 << 33, 3, N.LC_DTYPE_F16, 0.0) == (N.LC_NOT_SUPPORTED, 0)
    assert size(1, 4, 1, 1, N.LC_DTYPE_F16, 0.0) == (0, 0)
    st, n = size(1, 4, 1, 900, N.LC_DTYPE_F16, 0.0)  # long tables are split
    assert st == 0 and n > 0 and n % (4 * (64 + 2) * 4) == 0
    t = N.DeviceTensor(256, 256, 128, 64)
    r = ctypes.byref
    st = lib.lcKvCacheStore(r(pool), 1, 65, N.LC_DTYPE_F16, r(t), r(t), 256, 1, 1, None, None)
    assert st == N.LC_INVALID_VALUE and b"2 needed" in lib.lcGetLastErrorMessage()
    assert lib.lcKvCacheStore(r(pool), 1, 65, N.LC_DTYPE_F16, r(t), r(t), None, 2, 2, None, None) == N.LC_INVALID_VALUE
    empty = _pool(pages=0)
    assert lib.lcKvCacheStore(r(empty), 1, 65, N.LC_DTYPE_F16, r(t), r(t), 256, 2, 2, None,
                              None) == N.LC_INVALID_VALUE


def test_vit_norm_arguments():
    lib = N.load()
    assert lib.lcVitBlockSessionSetNorm(None, None, None, 1e-5) == N.LC_INVALID_VALUE


def test_host_tensors_are_refused_before_the_device():
    torch = pytest.importorskip("torch")
    x = torch.zeros(1, 1, 2, 16)
    with pytest.raises(ValueError, match="GPU memory"):
        lc.cross_attention(x, x, x)
    with pytest.raises(ValueError, match="GPU memory"):
        lc.layer_norm(x)
    with pytest.raises(ValueError, match="GPU memory"):
        lc.kv_cache_store(x, x, x, None, x, x, x, x)


@pytest.mark.skipif(lc.is_hip_available(), reason="checks the no-GPU behaviour")
def test_no_gpu_means_not_supported():
    x = np.zeros((1, 1, 2, 16), np.float32)
    with pytest.raises(RuntimeError, match="not supported"):
        lc.cross_attention(x, x, x)
    with pytest.raises(RuntimeError, match="not supported"):
        lc.layer_norm(x)
    out = ctypes.c_void_p(5)
    assert N.load().lcHipBackendStream(ctypes.byref(out)) == N.LC_NOT_SUPPORTED and not out.value
    assert N.load().lcHipBackendStream(None) == N.LC_INVALID_VALUE
