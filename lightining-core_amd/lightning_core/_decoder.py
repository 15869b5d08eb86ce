"""Operators of a decoder that reads an encoder's states: cross attention and
layer norm with their gradients, and an 8-bit paged cache of keys and values
with the attention that reads it.

Each function takes either torch tensors in the memory of the library's device
(results are torch tensors; the work is queued on torch's current stream of that
device, nothing is synchronised, and the call may be captured into a graph) or
numpy arrays (results are numpy arrays; the call returns when they are there).
Import torch before the library's first call: torch brings a HIP runtime of its
own, and a process in which the library has already started another one has no
device for torch.  The results carry no autograd history: a training step calls
the backward functions itself, and a tensor that requires a gradient is refused
unless the call is made under torch.no_grad().  Shapes, types and layouts that a
call does not take raise ValueError; a status of the library raises RuntimeError,
as everywhere in this package.
"""
from __future__ import annotations

import ctypes
import functools
import sys

import numpy as np

from . import _native as N
from ._core import _check, _lib

try:  # the compiled call helper, built next to the C library
    from ._addr import invoke as _invoke
except ImportError:  # not built: ctypes (slower, same result)
    _invoke = None

__all__ = ["cross_attention", "cross_attention_backward", "layer_norm", "layer_norm_backward", "kv_cache_store",
           "kv_cache_attention", "KV_PAGE_TOKENS"]

KV_PAGE_TOKENS = 64

_byref = ctypes.byref
_INT32_MOST = 2**31 - 1
_MOST_SCALE = 2.3e38  # times log2(e) it is still an fp32 number


def _is_torch(x) -> bool:
    torch = sys.modules.get("torch")
    return torch is not None and isinstance(x, torch.Tensor)


class _Torch:
    """Calls on torch tensors of one device.  One object per device: it keeps
    nothing of a call."""

    def __init__(self, torch, index):
        own = ctypes.c_int()
        _check(_lib().lcHipDeviceIndex(_byref(own)))
        if index != own.value:
            raise ValueError(f"the tensors are on cuda:{index}, the library computes on cuda:{own.value}")
        self.torch, self.index = torch, index
        self.device = torch.device("cuda", index)
        self._dtypes = {torch.float32: N.LC_DTYPE_F32, torch.bfloat16: N.LC_DTYPE_BF16,
                        torch.float16: N.LC_DTYPE_F16}
        self._types = {v: k for k, v in self._dtypes.items()}
        self._tensor = torch.Tensor
        self._empty = torch.empty
        self._tracking = torch.is_grad_enabled
        self._int32, self._float32 = torch.int32, torch.float32
        # The stream's handle without a Stream object around it (2 us a call less).
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._raw = raw or (lambda i: torch.cuda.current_stream(i).cuda_stream)

    @property
    def stream(self):
        return self._raw(self.index)

    def take(self, x, name):
        """x itself, when it is a tensor of this device."""
        if not isinstance(x, self._tensor):
            raise ValueError(f"{name} must be a torch tensor, as the other arguments are")
        if not x.is_cuda or x.get_device() != self.index:
            raise ValueError(f"{name} is on {x.device}, the other tensors on {self.device}")
        if x.requires_grad and self._tracking():
            raise ValueError(f"{name} requires a gradient that this call would not record: call it under "
                             "torch.no_grad() or with detached tensors, and the backward functions for gradients")
        return x

    def dtype(self, x, name):
        got = self._dtypes.get(x.dtype)
        if got is None:
            raise ValueError(f"{name} must be float32, bfloat16 or float16")
        return got

    def ints(self, x, name):
        self.take(x, name)
        if x.dtype is not self._int32:
            raise ValueError(f"{name} must be int32")
        return x

    @staticmethod
    def strides(x):
        return x.stride()

    @staticmethod
    def addr(x):
        return x.data_ptr()

    def empty(self, like, shape, dtype):
        return like.new_empty(shape, dtype=self._types[dtype])

    def empty_like(self, x):
        """x's type, shape and order of dimensions; the last one contiguous."""
        y = self.torch.empty_like(x)
        if y.stride(-1) != 1 and y.shape[-1] > 1:
            y = self._empty(x.shape, dtype=x.dtype, device=self.device)
        return y

    def empty_contiguous(self, x):
        return self.torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)

    def codes(self, x, name):
        self.take(x, name)
        if x.dtype is not self.torch.uint8 and x.dtype is not self.torch.float8_e4m3fn:
            raise ValueError(f"{name} must be uint8 or float8_e4m3fn")
        if not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return x

    def scales(self, x, name):
        self.take(x, name)
        if x.dtype is not self._float32 or not x.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32")
        return x

    @staticmethod
    def is_contiguous(x):
        return x.is_contiguous()

    @staticmethod
    def writable(*tensors):
        """Tensors have no such mark."""

    def workspace(self, nbytes):
        """Scratch of a call, held by the caller until the call is queued: the
        allocator hands it out again only to work queued behind it on the same
        stream."""
        return self._empty(nbytes, dtype=self.torch.uint8, device=self.device) if nbytes else None

    def rows(self, x, name):
        """(row count, row stride) of x seen as rows of its last dimension."""
        if x.ndim == 2:
            return x.shape[0], x.stride(0)
        try:
            v = x.view(-1, x.shape[-1]) if x.numel() else x.reshape(0, x.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}'s leading dimensions must collapse to rows of one stride") from None
        return v.shape[0], v.stride(0)

    @staticmethod
    def finish(*results):
        return results

    def run(self, name, spec, args, names):
        """Calls the entry point (spec: csrc/pyaddr.c; names: its 't' arguments')."""
        if _invoke is None:
            return _run_ctypes(self, name, spec, args, names)
        entry = _entries.get(name)
        if entry is None:
            entry = _entries[name] = ctypes.cast(getattr(_lib(), name), ctypes.c_void_p).value
        status = _invoke(entry, spec, *args)
        if status:
            if status < 0:
                raise ValueError(f"{names.split()[-1 - status]}'s last dimension must be contiguous")
            _check(status)


_torch_calls = {}
_entries = {}  # entry point -> its address


def _run_ctypes(call, name, spec, args, names):
    """The same call through ctypes."""
    names = iter(names.split())
    got = []
    for kind, x in zip(spec, args):
        if kind == "t":
            got.append(_tensor4(call, x, next(names)))
        elif kind == "p":
            got.append(None if x is None else call.addr(x))
        else:
            got.append(x)
    _check(getattr(_lib(), name)(*got))


def _torch_call(x):
    if not x.is_cuda:
        raise ValueError("torch tensors must be in GPU memory (pass numpy arrays for host data)")
    index = x.get_device()
    call = _torch_calls.get(index)
    if call is None:
        call = _torch_calls[index] = _Torch(sys.modules["torch"], index)
    return call


class _Numpy:
    """A call on numpy arrays: inputs go to device memory of the call's own, the
    work runs on the library's stream, results come back before it returns."""

    _dtypes = {np.dtype(np.float32): N.LC_DTYPE_F32, np.dtype(np.float16): N.LC_DTYPE_F16}
    _types = {N.LC_DTYPE_F32: np.float32, N.LC_DTYPE_F16: np.float16}

    def __init__(self):
        self._bufs = {}   # id(array) -> (device address, array)
        s = ctypes.c_void_p()
        _check(_lib().lcHipBackendStream(_byref(s)))
        self.stream = s.value

    def __del__(self):
        self.close()

    def close(self):
        for addr, _ in self._bufs.values():
            _lib().lcFree(addr)
        self._bufs = {}

    def take(self, x, name):
        if _is_torch(x):
            raise ValueError(f"{name} must be a numpy array, as the other arguments are")
        x = np.asarray(x)
        if x.dtype not in self._dtypes:
            x = x.astype(np.float32)
        return np.ascontiguousarray(x)

    def dtype(self, x, name):
        return self._dtypes[x.dtype]

    def ints(self, x, name):
        if _is_torch(x):
            raise ValueError(f"{name} must be a numpy array, as the other arguments are")
        x = np.asarray(x)
        if x.dtype.kind not in "iu":
            raise ValueError(f"{name} must hold integers")
        if x.dtype.itemsize > 2 and x.dtype != np.int32:
            # Numbers past 32 bits stay past every length and every pool.
            x = np.minimum(x, _INT32_MOST)
            if x.dtype.kind == "i":
                x = np.maximum(x, -_INT32_MOST)
        return np.ascontiguousarray(x, dtype=np.int32)

    def strides(self, x):
        return tuple(s // x.itemsize for s in x.strides)

    def _malloc(self, nbytes):
        p = ctypes.c_void_p()
        _check(_lib().lcMalloc(_byref(p), nbytes))
        return p.value

    def addr(self, x):
        if x.size == 0:
            return None
        got = self._bufs.get(id(x))
        if got is None:
            p = self._malloc(x.nbytes)
            self._bufs[id(x)] = got = (p, x)
            _check(_lib().lcMemcpy(p, x.ctypes.data, x.nbytes, N.LC_MEMCPY_HOST_TO_DEVICE))
        return got[0]

    def empty(self, like, shape, dtype):
        return np.zeros(shape, self._types[dtype])

    def empty_like(self, x):
        return np.zeros(x.shape, x.dtype)

    empty_contiguous = empty_like

    def codes(self, x, name):
        if not isinstance(x, np.ndarray) or x.dtype != np.uint8 or not x.flags.c_contiguous:
            raise ValueError(f"{name} must be a contiguous uint8 array")
        return x

    def scales(self, x, name):
        if not isinstance(x, np.ndarray) or x.dtype != np.float32 or not x.flags.c_contiguous:
            raise ValueError(f"{name} must be a contiguous float32 array")
        return x

    def is_contiguous(self, x):
        return x.flags.c_contiguous

    @staticmethod
    def writable(*arrays):
        for x, name in arrays:
            if not x.flags.writeable:
                raise ValueError(f"{name} is written and read-only")

    def workspace(self, nbytes):
        return np.empty(nbytes, np.uint8) if nbytes else None

    def rows(self, x, name):
        n = x.shape[-1]
        return (x.size // n if n else 0), n

    def run(self, name, spec, args, names):
        _run_ctypes(self, name, spec, args, names)

    def finish(self, *results):
        _check(_lib().lcDeviceSynchronize())
        for x in results:
            if x is not None and x.size:
                _check(_lib().lcMemcpy(x.ctypes.data, self._bufs[id(x)][0], x.nbytes, N.LC_MEMCPY_DEVICE_TO_HOST))
        self.close()
        return results


def _call_of(first):
    return _torch_call(first) if _is_torch(first) else _Numpy()


class _Struct:
    """A ctypes structure and its address, which lives as long as this does."""

    __slots__ = ("kept", "at")

    def __init__(self, kept):
        self.kept, self.at = kept, ctypes.addressof(kept)


def _tensor4(call, x, name):
    """The library's view of a [batch, heads, rows, d] tensor."""
    st = call.strides(x)
    if st[3] != 1 and x.shape[3] > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return _byref(N.DeviceTensor(call.addr(x), st[0], st[1], st[2]))


def _same(x, shape, name):
    if x.shape != shape:
        raise ValueError(f"{name} has shape {tuple(x.shape)}, expected {tuple(shape)}")


def _four(x, name):
    if x.ndim != 4:
        raise ValueError(f"{name} must have four dimensions [batch, heads, length, head_dim]")
    return x.shape


def _scale(scale):
    """The library's convention: 0 for 1 / sqrt(head_dim)."""
    if scale is None:
        return 0.0
    # As fp32, which is what the library gets: 1e-46 would reach it as 0.
    got = ctypes.c_float(scale).value
    if got == 0.0 or not abs(got) < _MOST_SCALE:
        raise ValueError(f"scale must be a number other than zero that fp32 holds, below 2.3e38: {scale}")
    return got


def _lengths(call, x, batch):
    if x is None:
        return None
    x = call.ints(x, "kv_lengths")
    _same(x, (batch,), "kv_lengths")
    if not call.is_contiguous(x):
        raise ValueError("kv_lengths must be contiguous")
    return x


def _out(call, out, like, name):
    """The caller's output tensor, or a new one like `like`."""
    if out is None:
        return call.empty_like(like)
    if isinstance(call, _Numpy):
        if not isinstance(out, np.ndarray) or not out.flags.c_contiguous:
            raise ValueError(f"{name} must be a contiguous array")
        call.writable((out, name))
    else:
        out = call.take(out, name)
    if out.dtype != like.dtype:
        raise ValueError(f"{name} must have the inputs' type")
    _same(out, like.shape, name)
    return out


@functools.lru_cache(maxsize=1024)
def _xattn_plan(q_shape, k_shape, dtype, scale):
    """The configuration of a pair of shapes and its workspaces' sizes."""
    b, hq, sq, d = q_shape
    bk, hkv, sk, dk = k_shape
    if bk != b or dk != d:
        raise ValueError("q and k must agree in batch and head_dim")
    if hkv == 0 or hq % hkv:
        raise ValueError("q's heads must be a multiple of k's")
    cfg = N.CrossAttentionConfig(b, hq, hkv, sq, sk, d, dtype, scale, 1)
    got = []
    for backward in (0, 1):
        n = ctypes.c_size_t()
        _check(_lib().lcCrossAttentionWorkspaceSize(_byref(cfg), backward, _byref(n)))
        got.append(n.value)
    return _Struct(cfg), got[0], got[1]


def _xattn_inputs(call, q, k, v, scale):
    q, k, v = call.take(q, "q"), call.take(k, "k"), call.take(v, "v")
    shape = _four(k, "k")
    if v.shape != shape:
        _same(v, shape, "v")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k and v must have one type")
    return q, k, v, _xattn_plan(_four(q, "q"), shape, call.dtype(q, "q"), _scale(scale))


def cross_attention(q, k, v, kv_lengths=None, *, scale=None, return_lse=False, out=None):
    """softmax(scale q k^T) v over each batch row's first kv_lengths[b] keys.

    q [batch, heads, q_len, head_dim]; k, v [batch, kv_heads, kv_len, head_dim]
    with heads a multiple of kv_heads (consecutive query heads share one);
    float32, bfloat16 or float16; any strides with a contiguous last dimension.
    kv_lengths int32 [batch] (None: kv_len everywhere), held to [0, kv_len].
    scale defaults to 1 / sqrt(head_dim).  A row without keys gives zeros.
    16-bit types: the softmax runs in fp32, its probabilities are rounded to the
    type for the product with v.
    out, if given, receives the result; it must not share memory with k or v.
    Returns out like q, with return_lse also the log of each row's sum of
    exponentials, float32 [batch, heads, q_len] (-inf without keys).  No autograd
    history: cross_attention_backward gives the gradients.
    """
    call = _call_of(q)
    q, k, v, (cfg, nbytes, _) = _xattn_inputs(call, q, k, v, scale)
    lengths = _lengths(call, kv_lengths, q.shape[0])
    out = _out(call, out, q, "out")
    if out is k or out is v:
        raise ValueError("out must not be k or v")
    lse = call.empty(q, q.shape[:3], N.LC_DTYPE_F32) if return_lse else None
    ws = call.workspace(nbytes)
    call.run("lcCrossAttentionForward", "itttptppii", (cfg.at, q, k, v, lengths, out, lse, ws, nbytes, call.stream),
             "q k v out")
    got = call.finish(out, lse)
    return got if return_lse else got[0]


def cross_attention_backward(dout, q, k, v, out, lse, kv_lengths=None, *, scale=None):
    """Gradients (dq, dk, dv) of cross_attention for the gradient dout of its
    result.  out and lse are what cross_attention(..., return_lse=True) returned
    for the same q, k, v, kv_lengths and scale.  dk and dv are sums over the
    query heads that share a head, and zero past a row's length.  16-bit types:
    P and dS are rounded to the type for the products with dout, k and q (fp16
    scaled by powers of two, so that values of any size keep their precision).
    """
    call = _call_of(q)
    q, k, v, (cfg, _, nbytes) = _xattn_inputs(call, q, k, v, scale)
    dout, out, lse = call.take(dout, "dout"), call.take(out, "out"), call.take(lse, "lse")
    for x, name in ((dout, "dout"), (out, "out")):
        _same(x, q.shape, name)
        if x.dtype != q.dtype:
            raise ValueError(f"{name} must have q's type")
    _same(lse, q.shape[:3], "lse")
    if call.dtype(lse, "lse") != N.LC_DTYPE_F32 or not call.is_contiguous(lse):
        raise ValueError("lse must be contiguous float32")
    lengths = _lengths(call, kv_lengths, q.shape[0])
    dq, dk, dv = call.empty_like(q), call.empty_like(k), call.empty_like(v)
    ws = call.workspace(nbytes)
    call.run("lcCrossAttentionBackward", "itttttpptttpii",
             (cfg.at, dout, q, k, v, out, lse, lengths, dq, dk, dv, ws, nbytes, call.stream),
             "dout q k v out dq dk dv")
    return call.finish(dq, dk, dv)


@functools.lru_cache(maxsize=512)
def _ln_plan(*key):
    cfg = N.LayerNormConfig(*key, 1)
    n = ctypes.c_size_t()
    _check(_lib().lcLayerNormWorkspaceSize(_byref(cfg), _byref(n)))
    return _Struct(cfg), n.value


def _vector(call, x, n, dtype, name):
    """A weight-like vector of n values: (vector, its type)."""
    x = call.take(x, name)
    _same(x, (n,), name)
    if not call.is_contiguous(x):
        raise ValueError(f"{name} must be contiguous")
    wd = call.dtype(x, name)
    if wd != dtype and wd != N.LC_DTYPE_F32:
        raise ValueError(f"{name} must be float32 or of x's type")
    return x, wd


def _ln_rows(call, x, name):
    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name} must have a last dimension of at least one value")
    if x.shape[-1] > 1 and call.strides(x)[-1] != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return call.rows(x, name)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, return_stats=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x [..., n], float32, bfloat16 or float16, its leading dimensions rows of one
    stride; weight, bias [n] of x's type or float32 (both the same), or None.
    Returns y (contiguous, like x), with return_stats also mean and
    rstd = 1 / sqrt(var + eps), float32 [...].  No autograd history:
    layer_norm_backward gives the gradients.
    """
    call = _call_of(x)
    x = call.take(x, "x")
    rows, stride = _ln_rows(call, x, "x")
    n, dtype = x.shape[-1], call.dtype(x, "x")
    wd = None
    if weight is not None:
        weight, wd = _vector(call, weight, n, dtype, "weight")
    if bias is not None:
        bias, bd = _vector(call, bias, n, dtype, "bias")
        if wd is not None and bd != wd:
            raise ValueError("weight and bias must have one type")
        wd = bd
    cfg, _ = _ln_plan(rows, n, dtype, dtype if wd is None else wd, float(eps))
    y = call.empty_contiguous(x)
    mean = rstd = None
    if return_stats:
        mean, rstd = call.empty(x, x.shape[:-1], N.LC_DTYPE_F32), call.empty(x, x.shape[:-1], N.LC_DTYPE_F32)
    call.run("lcLayerNormForward", "ipipppippi",
             (cfg.at, x, stride, weight, bias, y, n, mean, rstd, call.stream), "")
    got = call.finish(y, mean, rstd)
    return got if return_stats else got[0]


def layer_norm_backward(dy, x, weight, mean, rstd, *, bias=None):
    """Gradients (dx, dweight, dbias) of layer_norm for the gradient dy of its
    result.  mean and rstd are what layer_norm(..., return_stats=True) returned.
    dweight and dbias are in weight's type; with weight None, dweight is None and
    so is dbias, unless the bias that layer_norm took alone is given (its values
    do not matter, dbias is of its type).
    """
    call = _call_of(x)
    x, dy = call.take(x, "x"), call.take(dy, "dy")
    rows, stride = _ln_rows(call, x, "x")
    _same(dy, x.shape, "dy")
    if dy.dtype != x.dtype:
        raise ValueError("dy must have x's type")
    _, dy_stride = _ln_rows(call, dy, "dy")
    n, dtype = x.shape[-1], call.dtype(x, "x")
    wd = dtype
    if weight is not None:
        weight, wd = _vector(call, weight, n, dtype, "weight")
    if bias is not None:
        bias, bd = _vector(call, bias, n, dtype, "bias")
        if weight is not None and bd != wd:
            raise ValueError("weight and bias must have one type")
        wd = bd
    mean, rstd = call.take(mean, "mean"), call.take(rstd, "rstd")
    for s, name in ((mean, "mean"), (rstd, "rstd")):
        _same(s, x.shape[:-1], name)
        if call.dtype(s, name) != N.LC_DTYPE_F32 or not call.is_contiguous(s):
            raise ValueError(f"{name} must be contiguous float32")
    cfg, nbytes = _ln_plan(rows, n, dtype, wd, 0.0)
    dx = call.empty_contiguous(x)
    dw = db = None
    if weight is not None:
        dw, db = call.empty_contiguous(weight), call.empty_contiguous(weight)
    elif bias is not None:
        db = call.empty_contiguous(bias)
    ws = call.workspace(nbytes)
    call.run("lcLayerNormBackward", "ipipippppipppii",
             (cfg.at, dy, dy_stride, x, stride, weight, mean, rstd, dx, n, dw, db, ws, nbytes, call.stream), "")
    return call.finish(dx, dw, db)


def _cache(call, k_pages, v_pages, k_scales, v_scales):
    """The library's view of a page pool, and its tensors."""
    kp, vp = call.codes(k_pages, "k_pages"), call.codes(v_pages, "v_pages")
    ks, vs = call.scales(k_scales, "k_scales"), call.scales(v_scales, "v_scales")
    if kp.ndim != 4 or kp.shape[2] != KV_PAGE_TOKENS:
        raise ValueError(f"k_pages must be shaped [pages, kv_heads, {KV_PAGE_TOKENS}, head_dim]")
    pages, heads, _, d = kp.shape
    _same(vp, (pages, heads, d, KV_PAGE_TOKENS), "v_pages")
    _same(ks, (pages, heads), "k_scales")
    _same(vs, (pages, heads), "v_scales")
    return N.KvCache(call.addr(kp), call.addr(vp), call.addr(ks), call.addr(vs), pages, heads, d, 1), (kp, vp, ks, vs)


def _table(call, block_table, batch):
    t = call.ints(block_table, "block_table")
    if t.ndim != 2 or t.shape[0] != batch:
        raise ValueError("block_table must be shaped [batch, pages of a sequence]")
    st = call.strides(t)
    if t.shape[1] > 1 and st[1] != 1:
        raise ValueError("block_table's rows must be contiguous")
    return t, st[0]


def kv_cache_store(k, v, block_table, kv_lengths, k_pages, v_pages, k_scales, v_scales):
    """Writes keys and values to the pages of an 8-bit cache, in place.

    k, v [batch, kv_heads, kv_len, head_dim] (float32, bfloat16 or float16, any
    strides with a contiguous last dimension); block_table int32
    [batch, at least kv_len / 64 rounded up]; kv_lengths int32 [batch] or None
    (kv_len everywhere).  The pool: k_pages [pages, kv_heads, 64, head_dim] and
    v_pages [pages, kv_heads, head_dim, 64] of e4m3 codes (uint8, or torch's
    float8_e4m3fn), k_scales and v_scales float32 [pages, kv_heads].  Row b's
    first kv_lengths[b] tokens go to the pages block_table[b] from their start,
    each page and head with a scale of max(amax / 448, 2^-126); the rest of its
    last page becomes zeros and no other page changes.  A NaN has no part in amax
    and stays one; an infinity makes its whole page NaN.  Pages outside the pool
    are not written.  Rows that name one page must bring the same tokens for it.
    """
    call = _call_of(k)
    k, v = call.take(k, "k"), call.take(v, "v")
    b, h, sk, d = _four(k, "k")
    _same(v, k.shape, "v")
    if k.dtype != v.dtype:
        raise ValueError("k and v must have one type")
    c, pool = _cache(call, k_pages, v_pages, k_scales, v_scales)
    if (h, d) != (c.kv_heads, c.head_dim):
        raise ValueError("k and the cache must agree in kv_heads and head_dim")
    call.writable(*zip(pool, ("k_pages", "v_pages", "k_scales", "v_scales")))
    lengths = _lengths(call, kv_lengths, b)
    t, stride = _table(call, block_table, b)
    call.run("lcKvCacheStore", "iiiittpiipi",
             (ctypes.addressof(c), b, sk, call.dtype(k, "k"), k, v, t, t.shape[1], stride, lengths, call.stream), "k v")
    call.finish(*pool)


@functools.lru_cache(maxsize=1024)
def _kv_plan(pages, kv_heads, d, b, hq, sq, width, dtype, scale):
    # The size does not depend on where the pool lies: any aligned base does.
    cache = N.KvCache(16, 16, 16, 16, pages, kv_heads, d)
    cfg = N.KvAttentionConfig(b, hq, sq, width, dtype, scale)
    n = ctypes.c_size_t()
    _check(_lib().lcKvCacheAttentionWorkspaceSize(_byref(cache), _byref(cfg), _byref(n)))
    return _Struct(cfg), n.value


def kv_cache_attention(q, k_pages, v_pages, k_scales, v_scales, block_table, kv_lengths=None, *, scale=None,
                       return_lse=False, out=None):
    """cross_attention over the first kv_lengths[b] tokens of the pages
    block_table[b] of an 8-bit cache (see kv_cache_store for its layout).

    q [batch, heads, q_len, head_dim], heads a multiple of the cache's;
    kv_lengths int32 [batch] (None: every token of the table's pages).  Made for
    few query rows, such as a decode step's.  A table entry outside the pool is
    not read; rows that would need it come out as NaN.  Returns as
    cross_attention does; there is no gradient.
    """
    call = _call_of(q)
    q = call.take(q, "q")
    b, hq, sq, d = _four(q, "q")
    c, _ = _cache(call, k_pages, v_pages, k_scales, v_scales)
    if c.head_dim != d:
        raise ValueError("q and the cache must agree in head_dim")
    if c.kv_heads == 0 or hq % c.kv_heads:
        raise ValueError("q's heads must be a multiple of the cache's")
    lengths = _lengths(call, kv_lengths, b)
    t, stride = _table(call, block_table, b)
    cfg, nbytes = _kv_plan(c.pages, c.kv_heads, d, b, hq, sq, t.shape[1], call.dtype(q, "q"), _scale(scale))
    out = _out(call, out, q, "out")
    lse = call.empty(q, q.shape[:3], N.LC_DTYPE_F32) if return_lse else None
    ws = call.workspace(nbytes)
    call.run("lcKvCacheAttention", "iitpiptppii",
             (ctypes.addressof(c), cfg.at, q, t, stride, lengths, out, lse, ws, nbytes, call.stream), "q out")
    got = call.finish(out, lse)
    return got if return_lse else got[0]
