"""Attention over a paged cache of keys and values: what a generating model needs between its q / k / v projections
(``KSLinearGroup``) and its output projection (``ksmm_cu_cache_append``, ``ksmm_cu_cache_attention``).

The reference's attention sees one image at a time and keeps nothing (src/ksmm_py/model/vit.py:434-489).
"""
from __future__ import annotations

import ctypes
import operator

import torch
from torch import nn
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import native as _native
from .interface import KSLinear, KSLinearGroup
from .kernel import _result, _stream_ptr, dtype_code, no_tangents

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_INT = 2 ** 31


def rotary_frequencies(pairs, base=10000.0, device="cuda"):
    """``base ** (-i / pairs)`` radians per token for pair i, in 64 bits: what ``cache_append`` rotates by."""
    return float(base) ** (-torch.arange(pairs, dtype=torch.float64, device=device) / max(pairs, 1))


class KVCache:
    """A pool of pages for the keys and values of many sequences.

    ``keys`` and ``values`` are (pages, heads, page_size, head_dim) in ``dtype``: the model's type, or
    ``torch.float8_e4m3fn`` with an fp32 scale for each token and head, ``key_scales`` and ``value_scales``, (pages, heads,
    page_size).  Which page holds what is the caller's: tables are arguments of the calls.  New pages hold zeros."""

    def __init__(self, pages, page_size, heads, head_dim, dtype: torch.dtype = torch.float16, device: str = "cuda"):
        if min(pages, page_size, heads, head_dim) <= 0:
            raise ValueError("pages, page_size, heads and head_dim are positive")
        if str(device) == "cpu":
            raise Exception("kernel expects device='cuda'.")
        dims = (int(pages), int(heads), int(page_size), int(head_dim))
        eight = dtype == torch.float8_e4m3fn
        keys, values = (torch.zeros(dims, dtype=torch.uint8 if eight else dtype, device=device) for _ in range(2))
        if eight:
            keys, values = keys.view(dtype), values.view(dtype)
        self._set(keys, values, *((torch.zeros(dims[:3], device=device) for _ in range(2)) if eight else (None, None)))

    @classmethod
    def of(cls, keys, values, key_scales=None, value_scales=None):
        """A cache in tensors that are there: (pages, heads, page_size, head_dim) with any strides but the last, which is 1
        (a pool whose pages are (page_size, heads, head_dim) is passed transposed)."""
        cache = cls.__new__(cls)
        cache._set(keys, values, key_scales, value_scales)
        return cache

    def _set(self, keys, values, key_scales, value_scales):
        eight = isinstance(keys, torch.Tensor) and keys.dtype == torch.float8_e4m3fn
        for name, t in (("keys", keys), ("values", values)):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape != keys.shape or t.dtype != keys.dtype \
                    or t.device != keys.device:
                raise ValueError("keys and values are (pages, heads, page_size, head_dim) tensors of one shape, type and device")
            if t.dtype not in _TYPES and not eight:
                raise TypeError(f"a cache holds float32, float16, bfloat16 or float8_e4m3fn, not {t.dtype}")
            if t.shape[3] != 1 and t.stride(3) != 1:
                raise ValueError(f"{name}: the elements of a head are not next to each other")
            if min(t.shape[1:]) == 0:
                raise ValueError("page_size, heads and head_dim are positive")
            if t.requires_grad:
                raise ValueError("a cache is not trained through")
        for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
            if not eight:
                if t is not None:
                    raise ValueError(f"{name} belong to a float8_e4m3fn cache")
            elif not isinstance(t, torch.Tensor) or t.shape != keys.shape[:3] or t.dtype != torch.float32 or t.device != keys.device:
                raise ValueError(f"{name} must be a float32 tensor of shape {tuple(keys.shape[:3])} on the cache's device")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales

    pages = property(lambda self: self.keys.shape[0])
    heads = property(lambda self: self.keys.shape[1])
    page_size = property(lambda self: self.keys.shape[2])
    head_dim = property(lambda self: self.keys.shape[3])
    dtype = property(lambda self: self.keys.dtype)
    device = property(lambda self: self.keys.device)

    def __repr__(self):
        return (f"KVCache(pages={self.pages}, page_size={self.page_size}, heads={self.heads}, head_dim={self.head_dim}, "
                f"dtype={self.dtype})")


def _indexes(name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.dim() != len(shape) \
            or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        shape = tuple("any" if n is None else n for n in shape)
        raise ValueError(f"{name} must be an int32 tensor of shape {shape} on {device}")
    return t if t.numel() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _heads(name, t, heads, cache, tokens, dtype):
    """A (tokens, heads, head_dim) tensor as the kernels take it."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device != cache.device:
        raise ValueError(f"{name} must be a CUDA tensor on the cache's device")
    if t.dtype not in _TYPES or (dtype is not None and t.dtype != dtype):
        raise TypeError(f"{name} is {t.dtype}: expected {dtype or 'float32, float16 or bfloat16'}")
    if cache.dtype not in (t.dtype, torch.float8_e4m3fn):
        raise TypeError(f"{name} is {t.dtype}, the cache {cache.dtype}")
    if t.dim() != 3 or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads) \
            or (tokens is not None and t.shape[0] != tokens):
        want = tuple("any" if n is None else n for n in (tokens, heads, cache.head_dim))
        raise ValueError(f"{name} must have shape {want}, got {tuple(t.shape)}")
    if t.shape[1] == 0 or t.shape[1] % cache.heads:
        raise ValueError(f"{t.shape[1]} heads of {name} do not share {cache.heads} key heads evenly")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: a cache is not trained through")
    if t.shape[0] >= _MAX_INT - 65536:
        raise ValueError(f"{name} has {t.shape[0]} tokens")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _tensors(*ts):
    return all(isinstance(t, torch.Tensor) for t in ts)


def _tensors_or_none(*ts):
    return all(t is None or isinstance(t, torch.Tensor) for t in ts)


def _changed(*ts):
    """What a caller gave to be written counts as changed in place: a graph that kept it for its backward pass then raises."""
    increment_version([t for t in ts if t is not None and not t.is_inference()])


def _strides(t, n):
    return (ctypes.c_int64 * n)(*t.stride()[:n])


def _cache_desc(cache, table, lengths, starts, tokens):
    """Checks the tables; returns the descriptor and the tensors that it points into."""
    if not isinstance(cache, KVCache):
        raise TypeError("cache must be a KVCache")
    if not cache.keys.is_cuda:
        raise ValueError("cache must be on a CUDA device")
    lengths = _indexes("lengths", lengths, (None,), cache.device)
    table = _indexes("table", table, (lengths.shape[0], None), cache.device)
    if starts is not None:
        starts = _indexes("starts", starts, (lengths.shape[0] + 1,), cache.device)
    elif lengths.shape[0] and tokens % lengths.shape[0]:
        raise ValueError(f"{tokens} tokens do not divide into {lengths.shape[0]} sequences")
    if tokens and not lengths.shape[0]:
        raise ValueError("tokens without sequences")
    if max(table.shape[1] * cache.page_size, cache.pages, cache.heads, lengths.shape[0] * cache.heads) >= _MAX_INT - 65536:
        raise ValueError("the cache or its table is too large")
    d = _lib.CacheDesc(
        keys=cache.keys.data_ptr(), values=cache.values.data_ptr(), key_strides=_strides(cache.keys, 3),
        value_strides=_strides(cache.values, 3), pages=cache.pages, page_size=cache.page_size, kv_heads=cache.heads,
        head_dim=cache.head_dim, cache_dtype=_lib.KSMM_F8E4M3 if cache.key_scales is not None else dtype_code(cache.dtype),
        table=table.data_ptr(), table_stride=table.stride(0), table_width=table.shape[1], lengths=lengths.data_ptr(),
        starts=None if starts is None else starts.data_ptr(), sequences=lengths.shape[0], tokens=tokens)
    if cache.key_scales is not None:
        d.key_scales, d.value_scales = cache.key_scales.data_ptr(), cache.value_scales.data_ptr()
        d.key_scale_strides, d.value_scale_strides = _strides(cache.key_scales, 3), _strides(cache.value_scales, 3)
    return d, (table, lengths, starts)


def _output(name, out, like, device):
    if out.shape != like.shape or out.dtype != like.dtype or out.device != device or (out.stride(2) != 1 and out.shape[2] != 1):
        raise ValueError(f"{name} must have shape {tuple(like.shape)}, type {like.dtype} and neighbouring elements")
    if out.requires_grad:
        raise ValueError(f"{name} requires a gradient")
    return out


def cache_append(cache, table, lengths, k, v, q=None, *, starts=None, frequencies=None, interleaved=False, q_out=None):
    """Stores new tokens' keys and values in a paged cache, rotated by their positions on the way.

    ``k`` and ``v`` are (tokens, cache.heads, head_dim) with any strides (a part of ``KSLinearGroup``'s output is taken as it
    is), ``q`` (tokens, heads, head_dim).  ``lengths[s]`` (int32) is sequence s's number of tokens *with* the new ones,
    ``table[s, i]`` (int32) the page of its tokens ``i * page_size ..``.  Sequence s has the rows ``starts[s] .. starts[s +
    1] - 1``, or tokens / sequences rows each without ``starts``; the last of n rows has position ``lengths[s] - 1``.

    ``frequencies`` (float64, up to head_dim / 2; ``rotary_frequencies``) rotates pair i of every head of k and q by
    ``position * frequencies[i]``: elements (i, i + pairs), or (2 i, 2 i + 1) with ``interleaved``; the rest of the head is
    taken as it is.  Returns the rotated q (in ``q_out`` if given, which may be q), or None without q.  Rows of no sequence are
    zero in a q that the call makes, and left alone in ``q_out``.  A token whose page is not in the pool is not stored."""
    if not isinstance(cache, KVCache):
        raise TypeError("cache must be a KVCache")
    if _native is not None and _tensors(table, lengths, k, v) and _tensors_or_none(q, starts, frequencies, q_out):
        # one call of the extension module; None where it is not for it (a wrong argument, another order of elements)
        done = _native.cache_append(cache.keys, cache.values, cache.key_scales, cache.value_scales, table, lengths, k, v, q, starts,
                                    frequencies, bool(interleaved), q_out)
        if done is not None:
            return None if done is False else _result(done)
    no_tangents(k, v, q)
    k = _heads("k", k, cache.heads, cache, None, None)
    v = _heads("v", v, cache.heads, cache, k.shape[0], k.dtype)
    desc, keep = _cache_desc(cache, table, lengths, starts, k.shape[0])
    d = _lib.CacheAppendDesc(cache=desc, k=k.data_ptr(), v=v.data_ptr(), k_strides=_strides(k, 2), v_strides=_strides(v, 2),
                             heads=cache.heads, dtype=dtype_code(k.dtype), interleaved=int(bool(interleaved)))
    if frequencies is not None:
        if not isinstance(frequencies, torch.Tensor) or frequencies.dtype != torch.float64 or frequencies.dim() != 1 \
                or frequencies.device != cache.device or 2 * frequencies.shape[0] > cache.head_dim:
            raise ValueError(f"frequencies must be a float64 tensor of up to {cache.head_dim // 2} elements on {cache.device}")
        frequencies = frequencies.contiguous()
        d.frequencies, d.pairs = frequencies.data_ptr(), frequencies.shape[0]
    out = None
    if q is not None:
        q = _heads("q", q, None, cache, k.shape[0], k.dtype)
        if q.shape[1] > 65535:
            raise ValueError(f"q has {q.shape[1]} heads")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else _output("q_out", q_out, q, cache.device)
        d.q, d.q_out, d.q_strides, d.q_out_strides = q.data_ptr(), out.data_ptr(), _strides(q, 2), _strides(out, 2)
        d.heads, d.clear_rest = q.shape[1], int(q_out is None)
    elif q_out is not None:
        raise ValueError("q_out without q")
    with torch.cuda.device(cache.device):
        _lib.check(_lib.load().ksmm_cu_cache_append(ctypes.byref(d), _stream_ptr(cache.device)))
    _changed(cache.keys, cache.values, cache.key_scales, cache.value_scales, q_out)
    return out


def cache_attention(q, cache, table, lengths, *, starts=None, scale=None, window=None, max_new=None, out=None):
    """Attention of new tokens over their sequences' caches: ``softmax(scale * q K^T) V`` over the keys at positions up to
    the token's own (and after ``position - window``), zeros where there are none.

    ``q`` is (tokens, heads, head_dim); heads is a multiple of cache.heads, whose key head ``h // (heads // cache.heads)``
    serves head h.  ``table``, ``lengths`` and ``starts`` as in ``cache_append``, whose call comes first.  ``scale`` defaults to
    ``head_dim ** -0.5``.  ``max_new``: an upper bound of one sequence's new tokens, where the caller knows one (it picks the
    kernels; more tokens are still computed, slowly).  Rows of no sequence are zero in a result that the call makes,
    and left alone in ``out``, which may be q.  Rows that need a page which is not in the pool are NaN.  Nothing learns
    through this call."""
    if not isinstance(cache, KVCache):
        raise TypeError("cache must be a KVCache")
    window, max_new = (None if n is None else operator.index(n) for n in (window, max_new))
    if window is not None and window <= 0 or max_new is not None and max_new <= 0:
        raise ValueError("window and max_new are positive")
    if _native is not None and _tensors(q, table, lengths) and _tensors_or_none(starts, out):
        done = _native.cache_attention(q, cache.keys, cache.values, cache.key_scales, cache.value_scales, table, lengths, starts,
                                       cache.keys.shape[3] ** -0.5 if scale is None else float(scale),
                                       0 if window is None else min(window, _MAX_INT),
                                       0 if max_new is None else min(max_new, _MAX_INT), out)
        if done is not None:
            return _result(done)
    no_tangents(q)
    q = _heads("q", q, None, cache, None, None)
    desc, keep = _cache_desc(cache, table, lengths, starts, q.shape[0])
    if q.shape[1] > 65535:
        raise ValueError(f"q has {q.shape[1]} heads")
    result = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else _output("out", out, q, cache.device)
    d = _lib.CacheAttentionDesc(
        cache=desc, q=q.data_ptr(), out=result.data_ptr(), q_strides=_strides(q, 2), out_strides=_strides(result, 2),
        window=0 if window is None else min(window, _MAX_INT), max_new=0 if max_new is None else min(max_new, _MAX_INT),
        scale=cache.head_dim ** -0.5 if scale is None else float(scale), heads=q.shape[1], dtype=dtype_code(q.dtype),
        clear_rest=int(out is None))
    lib = _lib.load()
    with torch.cuda.device(cache.device):
        size = lib.ksmm_cu_cache_attention_workspace_bytes(ctypes.byref(d))
        ws = torch.empty(size, dtype=torch.uint8, device=cache.device) if size else None
        _lib.check(lib.ksmm_cu_cache_attention(ctypes.byref(d), ws.data_ptr() if size else None, size, _stream_ptr(cache.device)))
    _changed(out)
    return result


class KSAttention(nn.Module):
    """Causal attention of a generating model with Kronecker-sparse projections: q, k and v from one input
    (``KSLinearGroup``), rotated and appended to a ``KVCache`` (``cache_append``), attention over it (``cache_attention``) and the
    output layer (``KSLinear``), whose last kernel adds the residual.  It serves prompts, single tokens and batches of
    both; nothing learns through it.  The reference swaps the same four projections for Kronecker-sparse layers
    (src/ksmm_py/model/get_vit.py:164-215) around an attention without a cache.

    ``patterns``: of q, and of k and v where ``kv_patterns`` is None; ``kv_patterns`` with fewer features out give
    fewer key heads (each ``heads * head_dim / features`` query heads share one).  ``rotary_base`` None: no rotation;
    ``rotary_dim``: the features of a head that are rotated (default all)."""

    def __init__(self, patterns, out_patterns, heads, kv_patterns=None, bias=True, algo="kernel", dtype: torch.dtype = torch.float16,
                 device: str = "cuda", rotary_base=10000.0, rotary_dim=None, interleaved: bool = False, window=None, scale=None):
        super().__init__()
        if dtype not in _TYPES:
            raise TypeError(f"attention runs in float32, float16 or bfloat16, not {dtype}")
        if heads <= 0 or (window is not None and window <= 0):
            raise ValueError("heads and window are positive")

        def features(p):
            return p[-1][0] * p[-1][1] * p[-1][3]

        wide = features(patterns)
        if wide % heads:
            raise ValueError(f"{wide} features do not divide into {heads} heads")
        self.heads, self.head_dim = int(heads), wide // heads
        narrow = wide if kv_patterns is None else features(kv_patterns)
        if narrow % self.head_dim or self.heads % max(narrow // self.head_dim, 1):
            raise ValueError(f"{narrow} features of keys are no part of {heads} heads of {self.head_dim}")
        self.kv_heads = narrow // self.head_dim
        rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if rotary_dim % 2 or not 0 <= rotary_dim <= self.head_dim:
            raise ValueError(f"rotary_dim={rotary_dim}: an even number up to {self.head_dim}")
        kw = dict(bias=bias, algo=algo, dtype=dtype, device=device)
        out_in = out_patterns[0][0] * out_patterns[0][2] * out_patterns[0][3]
        if out_in != wide:
            raise ValueError(f"the output layer takes {out_in} features, the heads have {wide}")
        if kv_patterns is None:
            self.qkv = KSLinearGroup([KSLinear(patterns, **kw) for _ in range(3)])
        else:
            self.q = KSLinear(patterns, **kw)
            self.kv = KSLinearGroup([KSLinear(kv_patterns, **kw) for _ in range(2)])
        self.out = KSLinear(out_patterns, **kw)
        self.rotary_base = rotary_base
        self.dtype, self.window, self.scale, self.interleaved = dtype, window, scale, bool(interleaved)
        frequencies = None if rotary_base is None else rotary_frequencies(rotary_dim // 2, rotary_base, device)
        self.register_buffer("frequencies", frequencies, persistent=False)

    def _apply(self, fn, recurse=True):
        # (a change of the layers' type leaves the frequencies in 64 bits; memory that is not filled, which to_empty gives, is
        # filled: no state dict holds them)
        before = self.frequencies
        super()._apply(fn, recurse)
        if before is not None:
            device = self.frequencies.device
            if before.is_meta:
                self.frequencies = rotary_frequencies(before.shape[0], self.rotary_base, device)
            elif device.type != "meta":
                self.frequencies = before.to(device)
        return self

    def new_cache(self, pages, page_size=64, eight=False):
        """A ``KVCache`` for this layer, in its type or (``eight``) in 8 bits."""
        device = next(self.out.parameters()).device
        return KVCache(pages, page_size, self.kv_heads, self.head_dim, torch.float8_e4m3fn if eight else self.dtype, device)

    def forward(self, x, cache, table, lengths, starts=None, max_new=None, residual=None):
        """x: (..., features), flattened to tokens in the order that ``starts`` counts; with (sequences, n, features) and no
        ``starts`` every sequence has n new tokens.  ``table``, ``lengths`` (with the new tokens), ``starts`` and ``max_new`` as in
        ``cache_attention``; ``residual``: a tensor of the result's shape that is added to it."""
        for name, t in (("x", x), ("residual", residual)):
            if t is not None and t.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"{name} requires a gradient: a cache is not trained through")
        flat = x.reshape(-1, x.shape[-1])
        tokens = flat.shape[0]
        if hasattr(self, "qkv"):
            q, k, v = self.qkv(flat)
        else:
            q = self.q(flat)
            k, v = self.kv(flat)
        q = q.view(tokens, self.heads, self.head_dim)
        k, v = (t.view(tokens, self.kv_heads, self.head_dim) for t in (k, v))
        q = cache_append(cache, table, lengths, k, v, q=q, starts=starts, frequencies=self.frequencies, interleaved=self.interleaved)
        a = cache_attention(q, cache, table, lengths, starts=starts, scale=self.scale, window=self.window, max_new=max_new)
        wide, out = self.heads * self.head_dim, self.out.out_size
        y = self.out(a.view(tokens, wide), residual=None if residual is None else residual.reshape(tokens, out))
        return y.view(*x.shape[:-1], out)

    def extra_repr(self):
        return "heads={}, kv_heads={}, head_dim={}, window={}, interleaved={}".format(
            self.heads, self.kv_heads, self.head_dim, self.window, self.interleaved)
