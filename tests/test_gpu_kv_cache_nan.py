"""NaN and infinities among the values that enter the 8-bit cache."""
import math

import pytest
import torch

from gpu_util import require_hip

pytestmark = pytest.mark.gpu

PAGE, H, D = 64, 2, 32


@pytest.fixture(scope="module")
def lc():
    return require_hip()


def _pool(pages):
    return [torch.zeros((pages, H, PAGE, D), dtype=torch.uint8, device="cuda"),
            torch.zeros((pages, H, D, PAGE), dtype=torch.uint8, device="cuda"),
            torch.zeros((pages, H), device="cuda"), torch.zeros((pages, H), device="cuda")]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_one_bad_value(lc, dtype, value):
    gen = torch.Generator()
    gen.manual_seed(3)
    k, v = (torch.randn((1, H, 128, D), generator=gen).to(dtype).cuda() for _ in range(2))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    good = _pool(2)
    k0, v0 = k.clone(), v.clone()
    k0[0, 1, 70, 5], v0[0, 0, 3, 7] = 0, 0  # what the rest of the pages is to be
    lc.kv_cache_store(k0, v0, table, None, *good)
    k[0, 1, 70, 5], v[0, 0, 3, 7] = value, value
    pool = _pool(2)
    lc.kv_cache_store(k, v, table, None, *pool)
    # K's value lies in page 0 (the second), head 1; V's in page 1 (the first), head 0
    for i, (page, head, at) in ((0, (0, 1, (6, 5))), (1, (1, 0, (7, 3)))):
        code = int(pool[i][page, head][at])
        assert code & 0x7F == 0x7F
        rest, want = pool[i].clone(), good[i].clone()
        scales, want_scales = pool[i + 2].clone(), good[i + 2].clone()
        if math.isnan(value):
            rest[page, head][at] = want[page, head][at] = 0
        else:
            assert scales[page, head] == math.inf and (pool[i][page, head] & 0x7F == 0).sum() == PAGE * D - 1
            rest[page, head], want[page, head] = 0, 0
            scales[page, head] = want_scales[page, head] = 0
        assert torch.equal(rest, want) and torch.equal(scales, want_scales)
    q = torch.randn((1, H, 1, D), generator=gen).to(dtype).cuda()
    out = lc.kv_cache_attention(q, *pool, table)
    assert torch.isnan(out[0, 1]).all()  # a key's NaN reaches the whole row
    column = torch.isnan(out[0, 0, 0])
    assert column[7] and (column.all() if math.isinf(value) else column.sum() == 1)
    # rows that end before the bad key, or do not come so far, are as without it
    short = torch.tensor([64], dtype=torch.int32, device="cuda")
    got, want = (lc.kv_cache_attention(q, *p, table, short) for p in (pool, good))
    assert torch.equal(got[0, 1], want[0, 1])
