"""Decoder operators on torch tensors in device memory (include/speaksense.h, "decoder operators"): a paged key / value cache in 16 or 8 bits, attention of
new tokens over it, and filtered sampling of logits.

Calls launch on torch's current stream of the tensors' device and return at once; results and workspaces come from torch's allocator, so calls
can be captured into a graph.  Wrong arguments raise ValueError (or SpeakSenseError from the library) before anything is launched.  The operators serve: they
have no gradients, and tensors that ask for one are refused, inputs, settings and the cache's alike (use torch.no_grad() or detach()); so are forward-mode duals."""
from __future__ import annotations

import ctypes as C
from numbers import Integral
from typing import NamedTuple

import torch      # before the library: both must share one HIP runtime, torch's, and the loader keeps the first
from torch.autograd import forward_ad

from . import binding

KV_SAME, KV_E4M3, KV_INT8 = 0, 1, 2
_KINDS = {"same": KV_SAME, "e4m3": KV_E4M3, "int8": KV_INT8, KV_SAME: KV_SAME, KV_E4M3: KV_E4M3, KV_INT8: KV_INT8}
_DUAL = forward_ad if hasattr(forward_ad, "_current_level") else NamedTuple("Always", [("_current_level", int)])(0)      # a level below 0: no duals anywhere
_DTYPES = {torch.bfloat16: binding.DTYPE_BF16, torch.float16: binding.DTYPE_F16, torch.float32: 3}


class _Cache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("page_stride", C.c_int64), ("scale_stride", C.c_int64),
                ("n_pages", C.c_int32), ("page_size", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32), ("dtype", C.c_int32), ("kind", C.c_int32)]


class _Batch(C.Structure):
    _fields_ = [("page_table", C.c_void_p), ("q_start", C.c_void_p), ("kv_len", C.c_void_p), ("table_stride", C.c_int64), ("n_seqs", C.c_int32),
                ("max_pages", C.c_int32), ("n_tokens", C.c_int32), ("max_new", C.c_int32), ("min_new", C.c_int32), ("max_len", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("p", C.c_void_p), ("row_stride", C.c_int64), ("head_stride", C.c_int64)]


class _Sample(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "u", "temperature", "top_k", "top_p", "min_p", "id", "p", "logprob", "n_kept")] + \
               [("row_stride", C.c_int64), ("n_rows", C.c_int32), ("n_vocab", C.c_int32), ("dtype", C.c_int32), ("reserved", C.c_int32)]


_L = None


def _lib():
    global _L
    if _L is None:
        L = binding.lib()
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        if len(runtimes) > 1:
            raise ImportError(f"two HIP runtimes in this process ({', '.join(sorted(runtimes))}): import torch before speaksense_amd loads its library")
        sizes = (L.ss_sizeof_kv_cache(), L.ss_sizeof_kv_batch(), L.ss_sizeof_kv_rows(), L.ss_sizeof_sample_rows_args())
        if sizes != tuple(C.sizeof(s) for s in (_Cache, _Batch, _Rows, _Sample)):
            raise ImportError(f"{binding.LIB_PATH}: operator structs of {sizes} bytes are not this module's -- rebuild the library")
        cp, bp, rp, vp, i32 = C.POINTER(_Cache), C.POINTER(_Batch), C.POINTER(_Rows), C.c_void_p, C.c_int32
        L.ss_kv_append.argtypes = [cp, bp, rp, rp, i32, vp]
        L.ss_kv_read.argtypes = [cp, bp, rp, rp, i32, vp]
        L.ss_kv_attention_workspace.argtypes = [cp, bp, i32]
        L.ss_kv_attention_workspace.restype = C.c_int64
        L.ss_kv_attention.argtypes = [cp, bp, rp, i32, C.c_float, i32, rp, vp, vp, C.c_int64, i32, vp]
        L.ss_sample_rows.argtypes = [C.POINTER(_Sample), i32, vp]
        _L = L
    return _L


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _on(t, device, name):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a tensor in device memory")
    _need(device is None or t.device == device, f"{name} is on {t.device}, expected {device}")


def _no_gradient(t, name):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this operator does not have")
    if _DUAL._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode gradient, which this operator does not have")


if hasattr(torch._C, "_cuda_getCurrentRawStream"):      # 0.1 us; the public way builds a Stream object for 2
    _stream = torch._C._cuda_getCurrentRawStream
else:
    def _stream(index):
        return torch.cuda.current_stream(index).cuda_stream


class KvCache:
    """One layer's paged cache over the caller's tensors: k, v [n_pages, n_kv_heads, page_size, head_dim] and, in 8 bits, k_scale, v_scale
    [n_pages, n_kv_heads, page_size].  A page is contiguous; pages may be strided (views k = pool[:, 0], v = pool[:, 1] of one pool).

    kind "same": tensors of `dtype`; "e4m3": uint8 (or float8_e4m3fn) codes with uint8 exponents; "int8": int8 codes with float32 scales.
    dtype: float16 or bfloat16, the type of new keys and values, queries and results (for kind "same" that of k)."""

    def __init__(self, k, v, k_scale=None, v_scale=None, *, kind="same", dtype=None):
        _need(kind in _KINDS, f"unknown kind {kind!r}: 'same', 'e4m3' or 'int8'")
        self.kind = _KINDS[kind]
        _on(k, None, "k")
        _on(v, k.device, "v")
        dtype = k.dtype if dtype is None and self.kind == KV_SAME else dtype
        _need(dtype in (torch.float16, torch.bfloat16), "dtype must be torch.float16 or torch.bfloat16")
        held = {KV_SAME: (dtype,), KV_E4M3: (torch.uint8, torch.float8_e4m3fn), KV_INT8: (torch.int8,)}[self.kind]
        _need(k.dtype in held and v.dtype == k.dtype, f"k and v must be {held[0]}, got {k.dtype} and {v.dtype}")
        _need(k.dim() == 4 and v.shape == k.shape, "k and v must be [n_pages, n_kv_heads, page_size, head_dim], alike")
        n, heads, page, dim = k.shape
        _need(all(t.stride()[2:] == (dim, 1) and (heads == 1 or t.stride(1) == page * dim) for t in (k, v)) and (n == 1 or k.stride(0) == v.stride(0)), "each page must be contiguous, k and v with one stride between pages")
        scales = None
        if self.kind == KV_SAME:
            _need(k_scale is None and v_scale is None, "a 16-bit cache has no scales")
        else:
            scales = torch.uint8 if self.kind == KV_E4M3 else torch.float32
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                _on(t, k.device, name)
                _need(t.dtype == scales and t.shape == k.shape[:3], f"{name} must be {scales} [n_pages, n_kv_heads, page_size]")
                _need(t.stride(2) == 1 and (heads == 1 or t.stride(1) == page) and (n == 1 or t.stride(0) == k_scale.stride(0)), "each page's scales must be contiguous, with one stride between pages")
        self.k, self.v, self.k_scale, self.v_scale, self.dtype, self.device, self.index = k, v, k_scale, v_scale, dtype, k.device, k.get_device()
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n, heads, page, dim
        self._real = [(t, name) for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)) if t is not None and t.is_floating_point()]
        # a cache of one page may be a view whose stride says nothing
        page_stride = k.stride(0) if n > 1 else heads * page * dim
        scale_stride = 0 if scales is None else k_scale.stride(0) if n > 1 else heads * page
        self._c = _Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if scales is not None else None, v_scale.data_ptr() if scales is not None else None,
                         page_stride, scale_stride, n, page, heads, dim, _DTYPES[dtype], self.kind)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, page_size, head_dim, *, kind="same", dtype=torch.float16, device="cuda"):
        """A cache over new tensors (contents undefined: rows behind a sequence's length are never used)."""
        _need(kind in _KINDS, f"unknown kind {kind!r}: 'same', 'e4m3' or 'int8'")
        kd = _KINDS[kind]
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        held = {KV_SAME: dtype, KV_E4M3: torch.uint8, KV_INT8: torch.int8}[kd]
        k, v = (torch.empty(shape, dtype=held, device=device) for _ in "kv")
        if kd == KV_SAME:
            return cls(k, v, kind=kind, dtype=dtype)
        s = [torch.empty(shape[:3], dtype=torch.uint8 if kd == KV_E4M3 else torch.float32, device=device) for _ in "kv"]
        return cls(k, v, *s, kind=kind, dtype=dtype)


class KvBatch:
    """The sequences of one step: page_table [n_seqs, max_pages], q_start [n_seqs + 1], kv_len [n_seqs] (int32, in device memory), and what the scheduler
    knows on the host: the token rows n_tokens, the longest span of new tokens max_new (kv_attention computes no more of a span), and optionally the shortest and the longest kv_len.
    The tensors may change between calls (a captured graph reads their contents at replay), the host's numbers belong to the object."""

    def __init__(self, page_table, q_start, kv_len, *, n_tokens, max_new, min_new=0, max_len=0):
        _on(page_table, None, "page_table")
        for name, t in (("page_table", page_table), ("q_start", q_start), ("kv_len", kv_len)):
            _on(t, page_table.device, name)
            _need(t.dtype == torch.int32, f"{name} must be int32")
        _need(page_table.dim() == 2 and q_start.dim() == 1 and kv_len.dim() == 1, "page_table is [n_seqs, max_pages], q_start [n_seqs + 1], kv_len [n_seqs]")
        n, pages = page_table.shape
        _need(kv_len.numel() == n and q_start.numel() == n + 1, f"{n} rows of page_table, {kv_len.numel()} lengths, {q_start.numel()} starts")
        _need((pages <= 1 or page_table.stride(1) == 1) and (n == 0 or (kv_len.is_contiguous() and q_start.is_contiguous())), "rows of page_table, q_start and kv_len must be contiguous")
        _need(all(isinstance(x, Integral) and 0 <= x < 1 << 31 for x in (n_tokens, max_new, min_new, max_len)), "n_tokens, max_new, min_new and max_len must be host integers in [0, 2^31)")
        n_tokens, max_new, min_new, max_len = int(n_tokens), int(max_new), int(min_new), int(max_len)      # numpy's too
        self.page_table, self.q_start, self.kv_len, self.device, self.index = page_table, q_start, kv_len, page_table.device, page_table.get_device()
        self.n_seqs, self.n_tokens, self.max_new = n, n_tokens, max_new
        stride = page_table.stride(0) if n > 1 else pages
        self._c = _Batch(page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), stride, n, pages, n_tokens, max_new, min_new, max_len)


def _rows(t, name, cache, batch, heads):
    """The C view of token rows [n_tokens, heads, head_dim]; `heads` None: any number."""
    if isinstance(t, torch.Tensor) and t.dtype is cache.dtype and t.get_device() == cache.index:
        if t.requires_grad or _DUAL._current_level >= 0:
            _no_gradient(t, name)
        shape = t.shape
        if len(shape) == 3 and shape[0] == batch.n_tokens and shape[2] == cache.head_dim and (heads is None or shape[1] == heads):
            row, head, element = t.stride()
            if element == 1:       # a stride over one row or one head says nothing
                return _Rows(t.data_ptr(), row if shape[0] > 1 else cache.head_dim * shape[1], head if shape[1] > 1 else cache.head_dim)
    _on(t, cache.device, name)
    _need(t.dtype == cache.dtype, f"{name} must be {cache.dtype}, got {t.dtype}")
    _need(t.dim() == 3 and t.shape[0] == batch.n_tokens and t.shape[2] == cache.head_dim and (heads is None or t.shape[1] == heads),
          f"{name} must be [{batch.n_tokens}, {'n_heads' if heads is None else heads}, {cache.head_dim}], got {list(t.shape)}")
    raise ValueError(f"the elements of a head of {name} must be contiguous")


def _same_device(cache, batch):
    _need(isinstance(cache, KvCache) and isinstance(batch, KvBatch), "expected a KvCache and a KvBatch")
    _need(batch.index == cache.index, "the batch and the cache are on different devices")
    for t, name in cache._real:
        if t.requires_grad or _DUAL._current_level >= 0:
            _no_gradient(t, name)


def kv_append(cache: KvCache, batch: KvBatch, k, v) -> None:
    """Write the new tokens' keys and values [n_tokens, n_kv_heads, head_dim] into their pages, in the cache's form (ss_kv_append)."""
    _same_device(cache, batch)
    kr, vr = _rows(k, "k", cache, batch, cache.n_kv_heads), _rows(v, "v", cache, batch, cache.n_kv_heads)
    binding._check(_lib().ss_kv_append(cache._c, batch._c, kr, vr, cache.index, _stream(cache.index)))


def kv_read(cache: KvCache, batch: KvBatch, out=None):
    """What the cache holds at the tokens' positions, as (k, v) [n_tokens, n_kv_heads, head_dim] (ss_kv_read).  out: a pair of tensors to fill; token
    rows that no sequence owns are left as they were (new tensors: undefined)."""
    _same_device(cache, batch)
    if out is None:
        out = tuple(torch.empty((batch.n_tokens, cache.n_kv_heads, cache.head_dim), dtype=cache.dtype, device=cache.device) for _ in "kv")
    k, v = out
    kr, vr = _rows(k, "out[0]", cache, batch, cache.n_kv_heads), _rows(v, "out[1]", cache, batch, cache.n_kv_heads)
    binding._check(_lib().ss_kv_read(cache._c, batch._c, kr, vr, cache.index, _stream(cache.index)))
    return k, v


def kv_attention(cache: KvCache, batch: KvBatch, q, *, scale=None, causal=True, out=None, return_lse=False):
    """Attention of the new tokens' queries q [n_tokens, n_heads, head_dim] over their sequences' cached keys (ss_kv_attention) -> [n_tokens, n_heads,
    head_dim], with return_lse also float32 [n_tokens, n_heads].  scale: head_dim ** -0.5 unless given.  causal False: every token sees all kv_len keys."""
    _same_device(cache, batch)
    L = _lib()
    qr = _rows(q, "q", cache, batch, None)
    heads = q.shape[1]
    if out is None:
        out = torch.empty((batch.n_tokens, heads, cache.head_dim), dtype=cache.dtype, device=cache.device)
    orow = _rows(out, "out", cache, batch, heads)
    lse = torch.empty((batch.n_tokens, heads), dtype=torch.float32, device=cache.device) if return_lse else None
    need = L.ss_kv_attention_workspace(cache._c, batch._c, heads)
    if need < 0:
        binding._check(int(need))
    work = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    binding._check(L.ss_kv_attention(cache._c, batch._c, qr, heads, cache.head_dim ** -0.5 if scale is None else float(scale), 1 if causal else 0, orow,
                                     lse.data_ptr() if return_lse else None, work.data_ptr() if need else None, need, cache.index, _stream(cache.index)))
    return (out, lse) if return_lse else out


class Sampled(NamedTuple):
    id: torch.Tensor          # int32 [n_rows]
    p: torch.Tensor           # float32: weight among the kept ids
    logprob: torch.Tensor     # float32: before the filters
    n_kept: torch.Tensor      # int32


def sample_rows(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None) -> Sampled:
    """One id per row of logits [n_rows, n_vocab] (float32, float16 or bfloat16) from uniform numbers u [n_rows] (float64): temperature, top-k, top-p and
    min-p per row (ss_sample_rows).  Each setting is a tensor [n_rows] (float32; top_k int32) on the device, or None for "off"."""
    _on(logits, None, "logits")
    _no_gradient(logits, "logits")
    dev, index = logits.device, logits.get_device()
    _need(logits.dtype in _DTYPES, f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    _need(logits.dim() == 2 and (logits.shape[1] <= 1 or logits.stride(1) == 1), "logits must be [n_rows, n_vocab] with contiguous rows")
    n, v = logits.shape
    ptr = [logits.data_ptr()]
    for name, t, dt in (("u", u, torch.float64), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                        ("min_p", min_p, torch.float32)):
        if t is None and name != "u":
            ptr.append(None)
            continue
        if not (isinstance(t, torch.Tensor) and t.get_device() == index and t.dtype is dt and t.shape == (n,) and t.is_contiguous()):
            _on(t, dev, name)
            raise ValueError(f"{name} must be {dt} [{n}], contiguous")
        if t.requires_grad or _DUAL._current_level >= 0:
            _no_gradient(t, name)
        ptr.append(t.data_ptr())
    whole, real = torch.empty((2, n), dtype=torch.int32, device=dev), torch.empty((2, n), dtype=torch.float32, device=dev)
    ids, kept = whole.unbind()
    p, logprob = real.unbind()
    w, f = whole.data_ptr(), real.data_ptr()
    a = _Sample(*ptr, w, f, f + 4 * n, w + 4 * n, logits.stride(0) if n > 1 else v, n, v, _DTYPES[logits.dtype], 0)
    binding._check(_lib().ss_sample_rows(a, index, _stream(index)))
    return Sampled(ids, p, logprob, kept)
