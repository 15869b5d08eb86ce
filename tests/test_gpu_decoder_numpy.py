"""Decoder operators on numpy arrays: what is written has to be writable."""
import numpy as np
import pytest

from gpu_util import require_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def test_read_only_outputs_are_refused(lc):
    rng = np.random.default_rng(2)
    q, k = (rng.standard_normal((1, 2, s, 32)).astype(np.float32) for s in (3, 70))
    out = np.full_like(q, 7.0)
    out.flags.writeable = False
    with pytest.raises(ValueError, match="out is written and read-only"):
        lc.cross_attention(q, k, k, out=out)
    assert (out == 7).all()
    good = np.empty_like(q)
    assert lc.cross_attention(q, k, k, out=good) is good
    table = np.array([[1, 0]])
    for i, name in enumerate(("k_pages", "v_pages", "k_scales", "v_scales")):
        pool = [np.zeros((2, 2, 64, 32), np.uint8), np.zeros((2, 2, 32, 64), np.uint8),
                np.zeros((2, 2), np.float32), np.zeros((2, 2), np.float32)]
        pool[i].flags.writeable = False
        with pytest.raises(ValueError, match=f"{name} is written and read-only"):
            lc.kv_cache_store(k, k, table, None, *pool)
        assert all((x == 0).all() for x in pool)
        for x in pool:
            x.flags.writeable = True
        lc.kv_cache_store(k, k, table, None, *pool)
        for x in pool:  # read, but not written
            x.flags.writeable = False
        assert np.isfinite(lc.kv_cache_attention(q, *pool, table, [70])).all()


def test_read_only_inputs_are_fine(lc):
    x = np.arange(24, dtype=np.float32).reshape(2, 12)
    x.flags.writeable = False
    assert lc.layer_norm(x).shape == x.shape
