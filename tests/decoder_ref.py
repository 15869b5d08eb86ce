"""64-bit references of cross attention, layer norm and the 8-bit cache, with
bounds on what the kernels' roundings may change, from the definition alone.

U[t]: half a step of type t relative to the value.  fp32 sums of n terms are off
by at most n 2^-24 of the sum of their magnitudes.
"""
import math

import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
F = 2.0**-24
# Half a step below the type's normal numbers, where it no longer shrinks with
# the value: fp16's smallest subnormal is 2^-24, bf16's and fp32's 2^-133, 2^-149
# (fp32 arithmetic may drop subnormals: the smallest normal number).
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126, torch.float32: 2.0**-126}


def _key_mask(lengths, sk, device):
    return torch.arange(sk, device=device).view(1, 1, 1, -1) < lengths.view(-1, 1, 1, 1)


def _expand(x, heads):
    return x.double().repeat_interleave(heads // x.shape[1], dim=1)


def _clean(x, lengths):
    """x with the rows past each length set to zero, whatever they hold."""
    on = torch.arange(x.shape[2], device=x.device).view(1, 1, -1, 1) < lengths.view(-1, 1, 1, 1)
    return torch.where(on, x.double(), torch.zeros((), dtype=torch.float64, device=x.device))


class Attention:
    """Forward and backward of one call in 64 bits, and the kernels' bounds."""

    def __init__(self, q, k, v, lengths=None, scale=None, p_terms=1):
        b, hq, sq, d = q.shape
        sk = k.shape[2]
        dev = q.device
        self.u = U[q.dtype]
        self.dtype = q.dtype
        lengths = torch.full((b,), sk, dtype=torch.int64, device=dev) if lengths is None else lengths.to(dev).long()
        self.lengths = lengths.clamp(0, sk)
        self.scale = scale if scale is not None else 1 / math.sqrt(d)
        self.q = q.double()
        self.hkv = k.shape[1]
        self.k = _expand(_clean(k, self.lengths), hq)
        self.v = _expand(_clean(v, self.lengths), hq)
        on = _key_mask(self.lengths, sk, dev)
        s = self.q @ self.k.transpose(-1, -2) * self.scale
        s = s.masked_fill(~on, -math.inf)
        self.lse = torch.logsumexp(s, -1)
        self.p = torch.where(on, torch.exp(s - torch.where(self.lse == -math.inf, 0.0, self.lse).unsqueeze(-1)), 0.0)
        self.out = self.p @ self.v
        # A score: d products and the scaling in fp32; a probability: twice the
        # scores' error (its own and the reference's), the exponential, and the
        # sum over the keys.
        size = (self.q.abs() @ self.k.abs().transpose(-1, -2)) * abs(self.scale)
        top = size.amax(-1, keepdim=True) if sk else torch.zeros_like(size[..., :1])
        lse = torch.where(self.lse == -math.inf, 0.0, self.lse).abs().unsqueeze(-1)
        self.g = (2 * (d + 4) * top + 2 * lse + sk + 16) * F
        # P rounded for the second product (16-bit types); its sum likewise.
        self.up = 0.0 if q.dtype == torch.float32 else self.u**p_terms

    def out_bound(self):
        return self.u * self.out.abs() + (2 * self.up + 2 * self.g) * (self.p @ self.v.abs()) \
            + TINY[self.dtype]

    def lse_bound(self):
        return (self.g.squeeze(-1) + 2 * self.up + F * self.lse.abs()).nan_to_num(0.0, 0.0, 0.0)

    def _heads(self, x):
        b, h, s, d = x.shape
        return x.view(b, self.hkv, h // self.hkv, s, d).sum(2)

    def backward(self, dout):
        """{name: (gradient, bound)}; `out` and `lse` came rounded from the forward."""
        do = dout.double()
        d = do.shape[-1]
        dp = do @ self.v.transpose(-1, -2)
        delta = (do * self.out).sum(-1, keepdim=True)
        one = (self.lengths <= 1).view(-1, 1, 1, 1)  # a softmax over one key is constant
        ds = torch.where(one, 0.0, self.p * (dp - delta))
        grads = {"dq": ds @ self.k * self.scale, "dk": self._heads(ds.transpose(-1, -2) @ self.q) * self.scale,
                 "dv": self._heads(self.p.transpose(-1, -2) @ do)}
        # dP and delta in fp32; delta from an `out` that was rounded and computed
        # with rounded probabilities; dS rounded to the type.
        e_dp = (d + 4) * F * (do.abs() @ self.v.abs().transpose(-1, -2))
        size = do.abs() * (self.p @ self.v.abs())
        e_delta = (self.u * (do * self.out).abs() + (2 * self.up + 2 * self.g + (d + 4) * F) * size).sum(
            -1, keepdim=True)
        rows = self.p.shape[-2] * (do.shape[1] // self.hkv)
        keys = self.p.shape[-1]
        ur = 0.0 if self.dtype == torch.float32 else self.u
        e_ds = self.p * ((self.g + ur) * (dp - delta).abs() + (1 + self.g + ur) * (e_dp + e_delta))
        # exp2 gives nothing below 2^-126, and so does a product there.
        e_ds = e_ds + 2.0**-126 * (1 + (dp - delta).abs())
        low = 0.0
        if self.dtype == torch.float16:
            # dS is rounded with dO scaled to at least 1/8 at its largest: below
            # fp16's normal numbers half a step is 2^-25 of that scale.
            low = 2.0**-25 * 8 * do.abs().amax()
        s = abs(self.scale)
        full = ds.abs()
        bounds = {
            "dq": s * (((e_ds + low) + (keys + 4) * F * full) @ self.k.abs()),
            "dk": s * self._heads((e_ds + low + (rows + 4) * F * full).transpose(-1, -2) @ self.q.abs()),
            "dv": self._heads((self.p * (self.g + self.up + (rows + 4) * F)).transpose(-1, -2) @ do.abs()),
        }
        # P below the normal numbers, for dV.
        bounds["dv"] = bounds["dv"] + TINY[self.dtype] * self._heads(
            torch.ones_like(self.p).transpose(-1, -2) @ do.abs())
        tiny = TINY[self.dtype]
        return {n: (grads[n], bounds[n] * 1.01 + self.u * grads[n].abs() + tiny) for n in grads}


def assert_within(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} for {tuple(ref.shape)}"
    if got.numel() == 0:
        return
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities differ"
    assert torch.isfinite(got[~inf]).all(), f"{what}: a value is not finite"
    off = torch.where(inf, torch.zeros_like(ref), (got - ref).abs() - bound)
    worst = off.max()
    at = int(off.argmax())
    ratio = ((got - ref).abs() / bound)[~inf].max().item() if (~inf).any() else 0.0
    print(f"[bound] {what}: {ratio:.3f} of it", flush=True)
    assert worst <= 0, (f"{what}: element {at} is {got.flatten()[at].item():.8g}, {ref.flatten()[at].item():.8g} "
                        f"expected, bound {bound.flatten()[at].item():.3g}")
