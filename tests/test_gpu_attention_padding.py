"""16-bit cross attention gradients of a row do not depend on how far the other
rows pad the batch: up to 128 keys of its own, delta comes from the probabilities.
"""
import pytest
import torch

from decoder_ref import U, Attention, assert_within
from gpu_util import require_hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lc():
    return require_hip()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("sq", [1, 50, 300])
def test_padding_changes_nothing(lc, dtype, d, sq):
    gen = torch.Generator()
    gen.manual_seed(d + sq)
    lens, keys, hq, hkv = [18, 2, 64, 1, 0, 128, 100], 128, 4, 2
    b = len(lens)
    q, dout = (torch.randn((b, hq, sq, d), generator=gen).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn((b, hkv, keys, d), generator=gen).to(dtype).cuda() for _ in range(2))
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def run(pad, longer):
        """The batch padded to `pad`, with a row that is that long when `longer`."""
        extra = 1 if longer else 0
        x = [torch.randn((b + extra, t.shape[1], n, d), generator=gen).to(dtype).cuda()
             for t, n in ((dout, sq), (q, sq), (k, pad), (v, pad))]
        for y, t in zip(x, (dout, q, k, v)):
            y[:b, :, :t.shape[2]] = t
        n = torch.cat([lengths, torch.tensor([pad] * extra, dtype=torch.int32, device="cuda")])
        print(f"[case] {dtype} d={d} sq={sq} padded to {pad}", flush=True)
        out, lse = lc.cross_attention(x[1], x[2], x[3], n, return_lse=True)
        dq, dk, dv = lc.cross_attention_backward(x[0], *x[1:], out, lse, n)
        torch.cuda.synchronize()
        assert (dk[:b, :, keys:] == 0).all() and (dv[:b, :, keys:] == 0).all()
        return dq[:b], dk[:b, :, :keys], dv[:b, :, :keys]

    near = run(keys, False)
    ref = Attention(q, k, v, lengths).backward(dout)
    for pad, longer in ((1000, False), (1000, True), (129, True)):
        far = run(pad, longer)
        # one tile of keys: dQ is the same sum of the same products
        one_tile = [i for i, n in enumerate(lens) if n <= 64]
        assert torch.equal(far[0][one_tile], near[0][one_tile])
        for name, x, y in zip(("dq", "dk", "dv"), far, near):
            want, bound = ref[name]
            assert_within(x, want, bound, name)
            # others are summed in another order in 32 bits: a result next to a
            # border between two of its type's numbers falls on either side
            off = (x.double() - y.double()).norm() / y.double().norm().clamp_min(1e-30)
            assert off < U[dtype] / 4, (name, off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lengths_that_change_between_replays(lc, dtype):
    """A captured pass takes delta by the lengths of the replay, on either side of 128."""
    gen = torch.Generator()
    gen.manual_seed(9)
    q, dout = (torch.randn((3, 4, 40, 64), generator=gen).to(dtype).cuda() for _ in range(2))
    k, v = (torch.randn((3, 2, 500, 64), generator=gen).to(dtype).cuda() for _ in range(2))
    lengths = torch.tensor([500, 500, 500], dtype=torch.int32, device="cuda")

    def run():
        out, lse = lc.cross_attention(q, k, v, lengths, return_lse=True)
        return (out, lse) + tuple(lc.cross_attention_backward(dout, q, k, v, out, lse, lengths))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for turn in ([128, 129, 0], [1, 500, 127], [130, 2, 128], [500, 500, 500], [0, 0, 0]):
        lengths.copy_(torch.tensor(turn))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), turn
        ref = Attention(q, k, v, lengths).backward(dout)
        for name, x in zip(("dq", "dk", "dv"), got[2:]):
            assert_within(x, *ref[name], f"{turn} {name}")
