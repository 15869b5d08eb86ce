"""Arguments of the decoder operators that name something other than they seem to
(CPU only)."""
import ctypes

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
