"""The operators of a decoder that reads an encoder's states, as cases to time and compare.

A case is a dict of plain values; its "op" says which operator a pass runs:

* xattn       cross attention: queries of one length against keys and values of another
* xattn_bwd   its gradients with respect to queries, keys and values
* ln          layer norm, with the row statistics that its backward pass needs
* ln_bwd      its gradients with respect to input, weight and bias
* store       an encoder's keys and values written to the pages of an 8-bit cache
* cached      attention of a few new tokens over that cache

Lengths: `sk` is the padded number of encoder states; "ragged" gives each batch row a length of its own ("even": all are
`sk`; "half": from `sk` down to its half; "empty": the same, and the last row has none at all).
Cache pages hold 64 tokens of one key/value head: keys [page, head, token, d] and values [page, head, d, token] as
e4m3, each with one fp32 scale for a page and head.
"""
import math
import os
import sys

import torch

own = False

PAGE = 64
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_GPU = "cuda"


def _lc():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lightining-core_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lightning_core

    return lightning_core


def listed():
    return [
        # One new caption token of one request against the 196 patch tokens of a 224-pixel image.
        {"name": "xattn_token_f16_h12_196", "op": "xattn", "dtype": "f16", "b": 1, "hq": 12, "hkv": 12, "sq": 1,
         "sk": 196, "d": 64, "ragged": "even", "layout": "bhsd"},
        # A long prompt against a longer document, padded batch, activations as the projections leave them.
        {"name": "xattn_bf16_2048x4096", "op": "xattn", "dtype": "bf16", "b": 4, "hq": 16, "hkv": 16, "sq": 2048,
         "sk": 4096, "d": 128, "ragged": "half", "layout": "bshd"},
        # Default-precision training of a small decoder with shared key/value heads, lengths off every tile.
        {"name": "xattn_bwd_f32_77x1000", "op": "xattn_bwd", "dtype": "f32", "b": 2, "hq": 8, "hkv": 2, "sq": 77,
         "sk": 1000, "d": 64, "ragged": "half", "layout": "bhsd"},
        # A training step's cross attention at full length, four query heads to a key/value head.
        {"name": "xattn_bwd_bf16_2048x1500", "op": "xattn_bwd", "dtype": "bf16", "b": 4, "hq": 16, "hkv": 4,
         "sq": 2048, "sk": 1500, "d": 128, "ragged": "even", "layout": "bshd"},
        # The norm before the vision block's projections: eight images' tokens.
        {"name": "ln_f16_1568x768", "op": "ln", "dtype": "f16", "wdtype": "f16", "rows": 1568, "n": 768},
        # A prefill's norm at the widest model size of the GEMM benchmark.
        {"name": "ln_bf16_32768x8192", "op": "ln", "dtype": "bf16", "wdtype": "bf16", "rows": 32768, "n": 8192},
        # Default-precision training, a width that no vector load divides.
        {"name": "ln_bwd_f32_1000x1030", "op": "ln_bwd", "dtype": "f32", "wdtype": "f32", "rows": 1000, "n": 1030},
        # A training step's norm: 16-bit activations, fp32 weights.
        {"name": "ln_bwd_bf16_16384x4096", "op": "ln_bwd", "dtype": "bf16", "wdtype": "f32", "rows": 16384,
         "n": 4096},
        # Eight images' patch tokens enter the cache when their requests arrive.
        {"name": "store_f16_b8_196", "op": "store", "dtype": "f16", "b": 8, "hkv": 12, "sk": 196, "d": 64,
         "ragged": "even", "layout": "bshd"},
        # Sixteen long documents enter the cache.
        {"name": "store_bf16_b16_4096", "op": "store", "dtype": "bf16", "b": 16, "hkv": 16, "sk": 4096, "d": 128,
         "ragged": "half", "layout": "bshd"},
        # A decode step of eight caption requests.
        {"name": "cached_f16_b8_196", "op": "cached", "dtype": "f16", "b": 8, "hq": 12, "hkv": 12, "sq": 1, "sk": 196,
         "d": 64, "ragged": "even", "layout": "bhsd"},
        # A decode step of a full batch over long documents, shared key/value heads.
        {"name": "cached_bf16_b32_8192", "op": "cached", "dtype": "bf16", "b": 32, "hq": 32, "hkv": 8, "sq": 1,
         "sk": 8192, "d": 128, "ragged": "half", "layout": "bhsd"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xattn", "xattn", "xattn_bwd", "xattn_bwd", "ln", "ln_bwd", "store", "cached", "cached"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("ln", "ln_bwd"):
        n = _log(rng, 32, 8192)
        rows = _log(rng, 1, max(1, (32768 * 8192 if op == "ln" else 16384 * 4096) // (2 * n)))
        rows = min(rows, 65536)
        return {"op": op, "dtype": dtype, "wdtype": rng.choice([dtype, "f32"]), "rows": rows, "n": n}
    ragged = rng.choice(["even", "half", "half", "empty"])
    layout = rng.choice(["bhsd", "bshd"])
    if op in ("store", "cached"):
        b = rng.randint(2 if ragged == "empty" else 1, 16)
        case = {"op": op, "dtype": dtype, "b": b, "hkv": rng.choice([1, 2, 4, 8, 12]), "sk": _log(rng, 1, 4096),
                "d": rng.choice([32, 48, 64, 80, 128]), "ragged": ragged, "layout": layout}
        if op == "cached":
            case["hq"] = case["hkv"] * rng.choice([1, 1, 2, 4, 8])
            case["sq"] = rng.choice([1, 1, 1, 2, 3, 5])
        return case
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
    d = rng.choice([32, 40, 48, 64, 64, 80, 96, 128, 128])
    sq, sk = _log(rng, 1, 2048), _log(rng, 1, 1500)
    b = rng.randint(2 if ragged == "empty" else 1, 4) if group < 4 else rng.randint(1, 2)
    return {"op": op, "dtype": dtype, "b": b, "hq": hkv * group, "hkv": hkv, "sq": sq, "sk": sk, "d": d,
            "ragged": ragged if b > 1 else "half", "layout": layout}


# --- inputs ---------------------------------------------------------------------

def _lengths(case):
    """The keys of each batch row; the same for every seed, so that a case's work is known."""
    b, sk, kind = case["b"], case["sk"], case["ragged"]
    if kind == "even":
        return [sk] * b
    got = [max(1, sk - (i * sk) // (2 * b)) for i in range(b)]
    if kind == "empty":
        got[-1] = 0
    return got


def _heads(gen, b, h, s, d, dtype, layout, scale=1.0):
    """[b, h, s, d] values; "bshd": a transposed view of rows that hold all heads."""
    if layout == "bshd":
        return (torch.randn((b, s, h, d), generator=gen, device=_GPU) * scale).to(dtype).transpose(1, 2)
    return (torch.randn((b, h, s, d), generator=gen, device=_GPU) * scale).to(dtype)


def _pages_of(lengths):
    return [-(-n // PAGE) for n in lengths]


def _block_table(case, lengths, gen):
    """Every sequence's pages, scattered over the pool; -1 where it has no more."""
    need = _pages_of(lengths)
    width = max(1, -(-case["sk"] // PAGE))
    order = torch.randperm(sum(need) + 3, generator=gen, device=_GPU).to(torch.int32)
    table = torch.full((case["b"], width), -1, dtype=torch.int32, device=_GPU)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def prepare(case, seed):
    gen = torch.Generator(device=_GPU)
    gen.manual_seed(seed)
    op, dtype = case["op"], _DT[case["dtype"]]
    s = {"case": case}
    if op in ("ln", "ln_bwd"):
        rows, n, wdtype = case["rows"], case["n"], _DT[case["wdtype"]]
        # a residual stream: rows of different size, a mean of their own
        x = torch.randn((rows, n), generator=gen, device=_GPU)
        x *= torch.rand((rows, 1), generator=gen, device=_GPU) * 3 + 0.3
        x += torch.randn((rows, 1), generator=gen, device=_GPU) * 0.5
        s["x"] = x.to(dtype)
        s["weight"] = (1 + 0.2 * torch.randn(n, generator=gen, device=_GPU)).to(wdtype)
        s["bias"] = (0.2 * torch.randn(n, generator=gen, device=_GPU)).to(wdtype)
        if op == "ln_bwd":
            s["dy"] = torch.randn((rows, n), generator=gen, device=_GPU).to(dtype)
            del x
            _, s["mean"], s["rstd"] = _plain_ln(s["x"], s["weight"], s["bias"])
        return s
    b, hkv, sk, d, layout = case["b"], case["hkv"], case["sk"], case["d"], case["layout"]
    lengths = _lengths(case)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=_GPU)
    if op in ("store", "cached"):
        s["table"], pages = _block_table(case, lengths, gen)
        if op == "store":
            s["k"] = _heads(gen, b, hkv, sk, d, dtype, layout, 2.0)
            s["v"] = _heads(gen, b, hkv, sk, d, dtype, layout)
            s["cache"] = {"k_pages": torch.zeros((pages, hkv, PAGE, d), dtype=torch.uint8, device=_GPU),
                          "v_pages": torch.zeros((pages, hkv, d, PAGE), dtype=torch.uint8, device=_GPU),
                          "k_scales": torch.zeros((pages, hkv), device=_GPU),
                          "v_scales": torch.zeros((pages, hkv), device=_GPU)}
        else:
            # what a store of normal keys and values leaves: amax 3.5 to 4.5 over a page of one head
            def codes(shape):
                x = torch.randn(shape, generator=gen, device=_GPU) * (448 / 4.5)
                return x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)

            s["q"] = _heads(gen, b, case["hq"], case["sq"], d, dtype, layout)
            s["cache"] = {"k_pages": codes((pages, hkv, PAGE, d)), "v_pages": codes((pages, hkv, d, PAGE)),
                          "k_scales": (3.5 + torch.rand((pages, hkv), generator=gen, device=_GPU)) / 448,
                          "v_scales": (3.5 + torch.rand((pages, hkv), generator=gen, device=_GPU)) / 448}
        for name in ("k_pages", "v_pages"):
            s["cache"][name] = s["cache"][name].view(torch.float8_e4m3fn)
        return s
    s["q"] = _heads(gen, b, case["hq"], case["sq"], d, dtype, layout)
    s["k"] = _heads(gen, b, hkv, sk, d, dtype, layout)
    s["v"] = _heads(gen, b, hkv, sk, d, dtype, layout)
    if op == "xattn_bwd":
        s["dout"] = _heads(gen, b, case["hq"], case["sq"], d, dtype, layout)
        s["out"], s["lse"] = _plain_xattn(s["q"], s["k"], s["v"], s["lengths"])
    return s


# --- the operators in their plain form ---------------------------------------------

def _shared(x, heads):
    """Key/value heads repeated for the query heads that share them, in 32 bits."""
    return x.float().repeat_interleave(heads // x.shape[1], dim=1)


def _plain_probabilities(q, k, lengths):
    """softmax(q k^T / sqrt(d)) over each row's keys (zero where there is none), and the log of its sum."""
    s = torch.matmul(q.float(), _shared(k, q.shape[1]).transpose(-1, -2)) / math.sqrt(q.shape[-1])
    hidden = torch.arange(k.shape[2], device=k.device) >= lengths.view(-1, 1, 1, 1)
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    return p / torch.where(total == 0, torch.ones_like(total), total), lse


def _without_hidden(x, lengths):
    hidden = torch.arange(x.shape[2], device=x.device).view(1, 1, -1, 1) >= lengths.view(-1, 1, 1, 1)
    return x.masked_fill(hidden, 0)


def _like(x, ref):
    """x in ref's type and strides."""
    return torch.empty_like(ref).copy_(x)


def _plain_xattn(q, k, v, lengths):
    p, lse = _plain_probabilities(q, k, lengths)
    out = torch.matmul(p, _shared(_without_hidden(v, lengths), q.shape[1]))
    return _like(out, q), lse


def _plain_xattn_bwd(dout, q, k, v, lengths):
    b, hkv, sk, d = k.shape
    k, v = _without_hidden(k, lengths), _without_hidden(v, lengths)
    p, _ = _plain_probabilities(q, k, lengths)
    do = dout.float()
    dp = torch.matmul(do, _shared(v, q.shape[1]).transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
    dq = torch.matmul(ds, _shared(k, q.shape[1]))
    dk = torch.matmul(ds.transpose(-1, -2), q.float()).view(b, hkv, -1, sk, d).sum(2)
    dv = torch.matmul(p.transpose(-1, -2), do).view(b, hkv, -1, sk, d).sum(2)
    return _like(dq, q), _like(dk, k), _like(dv, v)


def _plain_ln(x, weight, bias, eps=1e-5):
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    c = xf - mean
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    y = c * rstd * weight.float() + bias.float()
    return y.to(x.dtype), mean.squeeze(-1), rstd.squeeze(-1)


def _plain_ln_bwd(dy, x, weight, mean, rstd):
    g = dy.float()
    xh = (x.float() - mean.unsqueeze(-1)) * rstd.unsqueeze(-1)
    dw, db = (g * xh).sum(0), g.sum(0)
    g = g * weight.float()
    dx = rstd.unsqueeze(-1) * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw.to(weight.dtype), db.to(weight.dtype)


def _plain_store(x, lengths, table, pages, scales, transposed):
    b, h, sk, d = x.shape
    width = table.shape[1]
    full = torch.zeros((b, h, width * PAGE, d), device=x.device)
    full[:, :, :sk] = _without_hidden(x, lengths).float()
    full = full.view(b, h, width, PAGE, d).permute(0, 2, 1, 3, 4)
    scale = (full.abs().amax((-1, -2)) / 448).clamp_min(2.0 ** -126)
    codes = (full / scale.unsqueeze(-1).unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    used = torch.arange(width, device=x.device) * PAGE < lengths.view(-1, 1)
    at = table[used].long()
    codes = codes[used]
    pages.view(torch.uint8)[at] = codes.transpose(-1, -2) if transposed else codes
    scales[at] = scale[used]


def _plain_values(pages, scales, table, transposed):
    """A cache's values for each batch row: [b, h, width * PAGE, d]."""
    at = table.clamp_min(0).long()
    x = pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scales[at].unsqueeze(-1).unsqueeze(-1)
    if transposed:
        x = x.transpose(-1, -2)
    b, width, h, _, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, width * PAGE, d)


def _plain_cached(q, c, table, lengths):
    k = _plain_values(c["k_pages"], c["k_scales"], table, False)
    v = _plain_values(c["v_pages"], c["v_scales"], table, True)
    return _plain_xattn(q, k, v, lengths)


def run(s):
    op = s["case"]["op"]
    if own:
        lc = _lc()
        if op == "xattn":
            out, lse = lc.cross_attention(s["q"], s["k"], s["v"], s["lengths"], return_lse=True)
            return {"out": out, "lse": lse}
        if op == "xattn_bwd":
            return dict(zip(("dq", "dk", "dv"), lc.cross_attention_backward(
                s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["lengths"])))
        if op == "ln":
            return dict(zip(("y", "mean", "rstd"), lc.layer_norm(s["x"], s["weight"], s["bias"], return_stats=True)))
        if op == "ln_bwd":
            return dict(zip(("dx", "dweight", "dbias"), lc.layer_norm_backward(
                s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])))
        c = s["cache"]
        if op == "store":
            lc.kv_cache_store(s["k"], s["v"], s["table"], s["lengths"], c["k_pages"], c["v_pages"], c["k_scales"],
                              c["v_scales"])
            return c
        out, lse = lc.kv_cache_attention(s["q"], c["k_pages"], c["v_pages"], c["k_scales"], c["v_scales"],
                                         s["table"], s["lengths"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "xattn":
        return dict(zip(("out", "lse"), _plain_xattn(s["q"], s["k"], s["v"], s["lengths"])))
    if op == "xattn_bwd":
        return dict(zip(("dq", "dk", "dv"), _plain_xattn_bwd(s["dout"], s["q"], s["k"], s["v"], s["lengths"])))
    if op == "ln":
        return dict(zip(("y", "mean", "rstd"), _plain_ln(s["x"], s["weight"], s["bias"])))
    if op == "ln_bwd":
        return dict(zip(("dx", "dweight", "dbias"), _plain_ln_bwd(s["dy"], s["x"], s["weight"], s["mean"],
                                                                  s["rstd"])))
    if op == "store":
        c = s["cache"]
        _plain_store(s["k"], s["lengths"], s["table"], c["k_pages"], c["k_scales"], False)
        _plain_store(s["v"], s["lengths"], s["table"], c["v_pages"], c["v_scales"], True)
        return c
    return dict(zip(("out", "lse"), _plain_cached(s["q"], s["cache"], s["table"], s["lengths"])))


# --- what a pass cannot do without ----------------------------------------------------

def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    e = size[case["dtype"]]
    if op in ("ln", "ln_bwd"):
        rows, n, we = case["rows"], case["n"], size[case["wdtype"]]
        if op == "ln":
            return {"bytes": 2 * rows * n * e + 2 * n * we + 8 * rows, "flops": 8 * rows * n}
        return {"bytes": 3 * rows * n * e + 3 * n * we + 8 * rows, "flops": 14 * rows * n}
    b, hkv, d = case["b"], case["hkv"], case["d"]
    keys = sum(_lengths(case))
    if op == "store":
        pages = sum(_pages_of(_lengths(case)))
        return {"bytes": 2 * keys * hkv * d * e + 2 * pages * hkv * (PAGE * d + 4) + 4 * pages,
                "flops": 4 * keys * hkv * d}
    hq, sq = case["hq"], case["sq"]
    rows = b * hq * sq
    if op == "cached":
        pages = sum(_pages_of(_lengths(case)))
        return {"bytes": 2 * keys * hkv * d + 8 * pages * hkv + 4 * pages + 2 * rows * d * e + 4 * rows,
                "flops": 4 * keys * hq * sq * d}
    if op == "xattn":
        return {"bytes": 2 * keys * hkv * d * e + 2 * rows * d * e + 4 * rows, "flops": 4 * keys * hq * sq * d}
    # q, dout, out read and dq written; keys and values read, their gradients written for every padded row
    return {"bytes": 4 * rows * d * e + 4 * rows + 2 * keys * hkv * d * e + 2 * b * case["sk"] * hkv * d * e,
            "flops": 10 * keys * hq * sq * d}


# --- the operators' values in 64 bits -----------------------------------------------------

def _exact_rows(q, k, scale):
    """One head of one batch row, all its keys visible: probabilities and log sum."""
    s = (q @ k.t()) * scale
    return torch.softmax(s, 1), torch.logsumexp(s, 1)


def _exact_xattn(q, keys_of, hkv, lengths):
    b, hq, sq, d = q.shape
    out = torch.zeros((b, hq, sq, d), dtype=torch.float64, device=q.device)
    lse = torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lengths):
        for h in range(hkv if n else 0):
            k, v = keys_of(i, h, n)
            for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                p, lse[i, j] = _exact_rows(q[i, j].double(), k, d ** -0.5)
                out[i, j] = p @ v
    return {"out": out, "lse": lse}


def _exact_codes(x):
    """x (64 bits, at most 448 + rounding) to the nearest e4m3 value, ties to even."""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(a / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("ln", "ln_bwd"):
        n = case["n"]
        y, mean, rstd, dx = [], [], [], []
        w = s["weight"].double()
        dw = torch.zeros(n, dtype=torch.float64, device=_GPU)
        db = torch.zeros_like(dw)
        for r in range(0, case["rows"], 4096):
            x = s["x"][r:r + 4096].double()
            var, mu = torch.var_mean(x, 1, correction=0, keepdim=True)
            sigma = torch.sqrt(var + 1e-5)
            hat = (x - mu) / sigma
            if op == "ln":
                y.append(hat * w + s["bias"].double())
                mean.append(mu[:, 0])
                rstd.append(1 / sigma[:, 0])
                continue
            g = s["dy"][r:r + 4096].double()
            dw += torch.einsum("rn,rn->n", g, hat)
            db += g.sum(0)
            a = g * w
            dx.append((a - (a.sum(1, keepdim=True) + hat * (a * hat).sum(1, keepdim=True)) / n) / sigma)
        if op == "ln":
            return {"y": torch.cat(y), "mean": torch.cat(mean), "rstd": torch.cat(rstd)}
        return {"dx": torch.cat(dx), "dweight": dw, "dbias": db}
    lengths = _lengths(case)
    hkv, d = case["hkv"], case["d"]
    if op == "xattn":
        return _exact_xattn(s["q"], lambda i, h, n: (s["k"][i, h, :n].double(), s["v"][i, h, :n].double()), hkv,
                            lengths)
    if op == "xattn_bwd":
        q, k, v, do = (s[x] for x in ("q", "k", "v", "dout"))
        dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=_GPU) for x in (q, k, v))
        group, scale = case["hq"] // hkv, d ** -0.5
        for i, n in enumerate(lengths):
            for j in range(case["hq"] if n else 0):
                h = j // group
                qj, kj, vj, gj = q[i, j].double(), k[i, h, :n].double(), v[i, h, :n].double(), do[i, j].double()
                p, _ = _exact_rows(qj, kj, scale)
                dv[i, h, :n] += p.t() @ gj
                dp = gj @ vj.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[i, j] = ds @ kj
                dk[i, h, :n] += ds.t() @ qj
        return {"dq": dq, "dk": dk, "dv": dv}
    table = s["table"].cpu()
    c = s["cache"]
    if op == "cached":
        kp, vp = (c[x].view(torch.uint8) for x in ("k_pages", "v_pages"))

        def keys_of(i, h, n):
            at = table[i, :-(-n // PAGE)].long().to(_GPU)
            k = kp[at, h].view(torch.float8_e4m3fn).double() * c["k_scales"][at, h].double().view(-1, 1, 1)
            v = vp[at, h].view(torch.float8_e4m3fn).double() * c["v_scales"][at, h].double().view(-1, 1, 1)
            return k.reshape(-1, d)[:n], v.transpose(1, 2).reshape(-1, d)[:n]

        return _exact_xattn(s["q"], keys_of, hkv, lengths)
    got = {x: t.double() if x.endswith("scales") else t.float() for x, t in c.items()}
    for i, n in enumerate(lengths):
        for p in range(-(-n // PAGE)):
            at, m = int(table[i, p]), min(PAGE, n - p * PAGE)
            for x, transposed in (("k", False), ("v", True)):
                rows = s[x][i, :, p * PAGE:p * PAGE + m].double()
                scale = (rows.abs().amax((1, 2)) / 448).clamp_min(2.0 ** -126)
                full = torch.zeros((hkv, PAGE, d), device=_GPU)
                full[:, :m] = _exact_codes(rows / scale.view(-1, 1, 1)).float()
                got[x + "_scales"][at] = scale
                got[x + "_pages"][at] = full.transpose(1, 2) if transposed else full
    return got
