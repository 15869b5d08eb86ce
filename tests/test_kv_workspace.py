"""The workspace of cached attention (CPU only): key splits are for few blocks of
rows, and a call whose blocks fill the chip needs none."""
import ctypes

import pytest

from lightning_core import _native as N


def _bytes(b, hq, hkv, sq, pages, d=128):
    pool = N.KvCache(256, 256, 256, 256, 1 << 20, hkv, d)
    cfg = N.KvAttentionConfig(b, hq, sq, pages, N.LC_DTYPE_BF16, 0.0)
    n = ctypes.c_size_t()
    assert N.load().lcKvCacheAttentionWorkspaceSize(ctypes.byref(pool), ctypes.byref(cfg), ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("shape", [
    (16, 32, 8, 2048, 32),   # a prompt: this was 1.1 GB
    (16, 32, 8, 64, 64), (4, 32, 8, 512, 32, 64), (64, 32, 8, 1, 64), (128, 32, 8, 1, 4096), (1, 16, 16, 512, 900),
])
def test_blocks_that_fill_the_chip_are_not_split(shape):
    assert _bytes(*shape) == 0


@pytest.mark.parametrize("shape", [(32, 32, 8, 1, 128), (16, 8, 8, 1, 256), (1, 4, 2, 1, 900), (1, 1, 1, 1, 40)])
def test_few_blocks_over_long_tables_are(shape):
    b, hq, _, sq, pages = shape
    n = _bytes(*shape)
    row = b * hq * sq * (128 + 2) * 4
    assert n % row == 0 and 2 <= n // row <= min(64, pages)
