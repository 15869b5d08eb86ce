"""Decoder operators and torch's autograd: no call drops a gradient silently."""
import pytest
import torch

import lightning_core as lc

pytestmark = pytest.mark.gpu


def _leaf(*shape):
    return torch.randn(*shape, device="cuda", requires_grad=True)


def _calls():
    """Every function with a tensor that requires a gradient in each place that can."""
    q, k = torch.randn(1, 2, 3, 64, device="cuda"), torch.randn(1, 2, 9, 64, device="cuda")
    out, lse = lc.cross_attention(q, k, k, return_lse=True)
    x, w = torch.randn(5, 32, device="cuda"), torch.randn(32, device="cuda")
    y, mean, rstd = lc.layer_norm(x, w, w, return_stats=True)
    pool = [torch.zeros(1, 2, 64, 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
    pool += [torch.ones(1, 2, device="cuda") for _ in range(2)]
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    args = {lc.cross_attention: [q, k, k], lc.cross_attention_backward: [q, q, k, k, out, lse],
            lc.layer_norm: [x, w, w], lc.layer_norm_backward: [x, x, w, mean, rstd],
            lc.kv_cache_store: [k, k, table, None, *pool], lc.kv_cache_attention: [q, *pool, table]}
    for fn, a in args.items():
        for i, t in enumerate(a):
            if torch.is_tensor(t) and t.is_floating_point():
                yield fn, a[:i] + [t.clone().requires_grad_()] + a[i + 1:]


def test_tensors_that_require_a_gradient_are_refused():
    n = 0
    for fn, args in _calls():
        with pytest.raises(ValueError, match="requires a gradient"):
            fn(*args)
        with torch.no_grad():
            fn(*args)
        with torch.inference_mode():
            fn(*args)
        fn(*[a.detach() if torch.is_tensor(a) else a for a in args])
        n += 1
    assert n == 3 + 6 + 3 + 5 + 4 + 3
    torch.cuda.synchronize()


def test_an_output_of_the_caller_that_requires_a_gradient():
    q, k = torch.randn(1, 2, 3, 64, device="cuda"), torch.randn(1, 2, 9, 64, device="cuda")
    with pytest.raises(ValueError, match="out requires a gradient"):
        lc.cross_attention(q, k, k, out=_leaf(1, 2, 3, 64))


def test_values_of_a_graph_are_refused_too():
    """Not leaves alone: a value whose history leads to one."""
    x = _leaf(5, 32) * 2
    with pytest.raises(ValueError, match="x requires a gradient"):
        lc.layer_norm(x)
    with torch.no_grad():
        assert not lc.layer_norm(x).requires_grad
