"""Arguments of the decoder operators that name something other than they seem to
(CPU only)."""
import ctypes

import numpy as np
import pytest

from lightning_core import _decoder
from lightning_core import _native as N


def _size(scale):
    cfg = N.CrossAttentionConfig(1, 2, 1, 3, 9, 64, N.LC_DTYPE_F16, scale)
    n = ctypes.c_size_t(77)
    return N.load().lcCrossAttentionWorkspaceSize(ctypes.byref(cfg), 0, ctypes.byref(n)), n.value


@pytest.mark.parametrize("scale", [0, 0.0, 1e-46, -1e-46, 1e39, -1e39, 3e38, float("nan"), float("inf")])
def test_scales_that_fp32_does_not_hold(scale):
    """0 stands for 1 / sqrt(head_dim) in the library: no other number may reach it as 0."""
    with pytest.raises(ValueError, match="scale"):
        _decoder._scale(scale)
    held = ctypes.c_float(scale).value
    if held:
        assert _size(held) == (N.LC_INVALID_VALUE, 0)


def test_scales_reach_the_library_as_they_are():
    assert _decoder._scale(None) == 0.0
    for scale in (1.0, -2.5, 0.1, 1e-45, 2.2e38):
        assert _decoder._scale(scale) == ctypes.c_float(scale).value != 0
        assert _size(_decoder._scale(scale))[0] == 0


@pytest.mark.parametrize("kind", ["i1", "u1", "i2", "u2", "i4", "u4", "i8", "u8"])
def test_integers_of_numpy_arrays_keep_their_order(kind):
    """What passes 32 bits is held to them, not wrapped: a length of 2^32 + 1 is not 1."""
    info = np.iinfo(kind)
    values = [v for v in (0, 1, 5, 100, 2**31 - 1, 2**31, 2**32, 2**32 + 1, 2**63 - 1, 2**64 - 1, -1, -7, -2**31,
                          -2**32 + 3, -2**63) if info.min <= v <= info.max]
    got = _decoder._Numpy.ints(None, np.array(values, dtype=kind), "kv_lengths")
    assert got.dtype == np.int32
    for v, g in zip(values, got.tolist()):
        assert g == max(min(v, 2**31 - 1), -2**31) or (v < -2**30 and g < -2**30)
    assert _decoder._Numpy.ints(None, [3, 4], "kv_lengths").tolist() == [3, 4]
    for bad in ([1.5], [True], ["a"]):
        with pytest.raises(ValueError, match="integers"):
            _decoder._Numpy.ints(None, np.array(bad), "kv_lengths")


@pytest.mark.parametrize("strides,shape,fits", [
    ((384, 192, 64), (2, 2, 3), True),      # batch, heads, rows in order
    ((384, 64, 128), (2, 2, 3), True),      # rows that hold both heads
    ((64, 768, 128), (2, 2, 3), True),      # the batch innermost
    ((400, 196, 65), (2, 2, 3), True),      # padding behind rows and heads
    ((64, 64, 128), (2, 2, 3), False),      # two batch rows in the heads' place
    ((192, 192, 64), (2, 2, 3), False),     # batch and heads one apart
    ((128, 192, 64), (2, 2, 3), False),     # a head reaches into the next
    ((384, 192, 63), (2, 2, 3), False),
    ((0, 0, 0), (1, 1, 1), True),           # nothing to step over
    ((0, 64, 128), (1, 2, 3), True),
    ((0, 64, 128), (2, 2, 3), False),
])
def test_written_tensors_do_not_overlap_themselves(strides, shape, fits):
    """Checked before the device is opened: a tensor that fits gets as far as the
    next one, which has no base."""
    lib = N.load()
    b, h, s = shape
    cfg = N.CrossAttentionConfig(b, h, h, s, s, 64, N.LC_DTYPE_F16, 0.0)
    r = ctypes.byref
    ok, none = N.DeviceTensor(256, h * s * 64, s * 64, 64), N.DeviceTensor(None, h * s * 64, s * 64, 64)
    dq = N.DeviceTensor(256, *strides)
    assert lib.lcCrossAttentionBackward(r(cfg), r(ok), r(ok), r(ok), r(ok), r(ok), 256, None, r(dq), r(none), r(ok),
                                        None, 0, None) == N.LC_INVALID_VALUE
    message = lib.lcGetLastErrorMessage().decode()
    assert ("dk has values and a null base" in message) if fits else ("dq is written and has overlapping" in message)


def test_problems_past_a_launch_are_not_supported():
    """256 threads a (batch row, key/value head) pair, less than 2^32 in a launch."""
    lib = N.load()

    def attention(b, heads):
        cfg = N.CrossAttentionConfig(b, heads, heads, 1, 1, 16, N.LC_DTYPE_F16, 0.0)
        return lib.lcCrossAttentionWorkspaceSize(ctypes.byref(cfg), 0, ctypes.byref(ctypes.c_size_t()))

    def cached(b, heads):
        pool = N.KvCache(256, 256, 256, 256, 4, heads, 16)
        cfg = N.KvAttentionConfig(b, heads, 1, 1, N.LC_DTYPE_F16, 0.0)
        return lib.lcKvCacheAttentionWorkspaceSize(ctypes.byref(pool), ctypes.byref(cfg),
                                                   ctypes.byref(ctypes.c_size_t()))

    for call in (attention, cached):
        assert call((1 << 24) - 1, 1) == 0 and call((1 << 23) - 1, 2) == 0
        assert call(1 << 24, 1) == N.LC_NOT_SUPPORTED and call(1 << 22, 4) == N.LC_NOT_SUPPORTED
