"""What KVCache, cache_append, cache_attention and their C entry points refuse; no GPU."""
import ctypes

import pytest
import torch

import ksmm_b200 as kb
from ksmm_b200 import _lib

F8 = torch.float8_e4m3fn


def pool(dtype=torch.float16, shape=(3, 2, 16, 64)):
    return torch.zeros(shape).to(dtype)


def test_cache_arguments():
    with pytest.raises(Exception, match="cuda"):
        kb.KVCache(2, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        kb.KVCache(0, 16, 2, 64)
    with pytest.raises(ValueError, match="one shape"):
        kb.KVCache.of(pool(), pool(shape=(3, 2, 16, 32)))
    with pytest.raises(ValueError, match="one shape"):
        kb.KVCache.of(pool(), pool(torch.bfloat16))
    with pytest.raises(ValueError, match="one shape"):
        kb.KVCache.of(None, pool())
    with pytest.raises(TypeError):
        kb.KVCache.of(pool(torch.float64), pool(torch.float64))
    with pytest.raises(ValueError, match="next to each other"):
        kb.KVCache.of(pool().transpose(2, 3), pool().transpose(2, 3))
    with pytest.raises(ValueError, match="scales"):
        kb.KVCache.of(pool(F8), pool(F8))
    with pytest.raises(ValueError, match="scales"):
        kb.KVCache.of(pool(), pool(), torch.zeros(3, 2, 16), torch.zeros(3, 2, 16))
    with pytest.raises(ValueError, match="scales"):
        kb.KVCache.of(pool(F8), pool(F8), torch.zeros(3, 2, 16), torch.zeros(3, 2, 8))
    with pytest.raises(ValueError, match="trained"):
        kb.KVCache.of(pool().requires_grad_(), pool())
    c = kb.KVCache.of(pool(), pool())
    assert (c.pages, c.heads, c.page_size, c.head_dim, c.dtype) == (3, 2, 16, 64, torch.float16) and "pages=3" in repr(c)


def test_calls_on_host_tensors():
    cache = kb.KVCache.of(pool(), pool())
    x, n = torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kb.cache_attention(x, cache, n[:, None], n)
    with pytest.raises(ValueError, match="CUDA"):
        kb.cache_append(cache, n[:, None], n, x, x)
    with pytest.raises(TypeError, match="KVCache"):
        kb.cache_attention(x, pool(), n[:, None], n)


def descs(**kw):
    """Descriptors of both calls over host memory, which a refused call does not touch."""
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    cache = dict(keys=p, values=p, pages=4, page_size=16, kv_heads=2, head_dim=64, cache_dtype=_lib.KSMM_F16, table=p, table_stride=4,
                 table_width=4, lengths=p, sequences=2, tokens=2)
    call = dict(q=p, heads=4, dtype=_lib.KSMM_F16)
    for k, v in kw.items():
        (cache if k in cache or k in ("starts", "key_scales", "value_scales") else call)[k] = v
    c = _lib.CacheDesc(**cache)
    own = {k: v for k, v in call.items() if k in ("window", "max_new", "out")}
    both = {k: v for k, v in call.items() if k in ("q", "heads", "dtype")}
    rest = {k: v for k, v in call.items() if k not in own and k not in both}
    a = _lib.CacheAppendDesc(cache=c, **{**dict(k=p, v=p, q_out=p), **both, **rest})
    t = _lib.CacheAttentionDesc(cache=c, **{**dict(out=p, scale=1.0), **both, **own})
    a._keep = t._keep = buf
    return a, t


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=_lib.KSMM_F8E4M3), _lib.KSMM_ERR_UNSUPPORTED, b"float32"),
    (dict(cache_dtype=_lib.KSMM_BF16), _lib.KSMM_ERR_UNSUPPORTED, b"model's type"),
    (dict(cache_dtype=_lib.KSMM_F8E4M3), _lib.KSMM_ERR_BAD_ARGUMENT, b"scales"),
    (dict(head_dim=257), _lib.KSMM_ERR_UNSUPPORTED, b"256"),
    (dict(head_dim=0), _lib.KSMM_ERR_BAD_ARGUMENT, b"positive"),
    (dict(page_size=0), _lib.KSMM_ERR_BAD_ARGUMENT, b"positive"),
    (dict(kv_heads=3), _lib.KSMM_ERR_BAD_ARGUMENT, b"share"),
    (dict(heads=65536), _lib.KSMM_ERR_BAD_ARGUMENT, b"share"),
    (dict(pages=-1), _lib.KSMM_ERR_BAD_ARGUMENT, b"positive"),
    (dict(pages=2 ** 31), _lib.KSMM_ERR_BAD_ARGUMENT, b"pages"),
    (dict(tokens=-1), _lib.KSMM_ERR_BAD_ARGUMENT, b"sequences and tokens"),
    (dict(tokens=2 ** 31), _lib.KSMM_ERR_BAD_ARGUMENT, b"sequences and tokens"),
    (dict(tokens=3), _lib.KSMM_ERR_BAD_ARGUMENT, b"divide"),
    (dict(sequences=0), _lib.KSMM_ERR_BAD_ARGUMENT, b"without sequences"),
    (dict(table_width=2 ** 28), _lib.KSMM_ERR_BAD_ARGUMENT, b"table_width"),
    (dict(lengths=None), _lib.KSMM_ERR_BAD_ARGUMENT, b"null"),
    (dict(table=None), _lib.KSMM_ERR_BAD_ARGUMENT, b"null"),
    (dict(keys=None), _lib.KSMM_ERR_BAD_ARGUMENT, b"null"),
])
def test_both_calls_refuse(kw, status, text):
    lib = _lib.load()
    before = lib.ksmm_cu_launch_count()
    a, t = descs(**kw)
    assert lib.ksmm_cu_cache_append(ctypes.byref(a), None) == status and text in lib.ksmm_cu_last_error()
    assert lib.ksmm_cu_cache_attention(ctypes.byref(t), None, 0, None) == status and text in lib.ksmm_cu_last_error()
    assert lib.ksmm_cu_cache_attention_workspace_bytes(ctypes.byref(t)) == 0
    assert lib.ksmm_cu_launch_count() == before


def test_each_call_refuses():
    lib = _lib.load()
    for kw, text in ((dict(k=None), b"null"), (dict(v=None), b"null"), (dict(q_out=None), b"null"), (dict(pairs=4), b"null"),
                     (dict(pairs=33), b"pairs"), (dict(pairs=-1), b"pairs")):
        a, _ = descs(**kw)
        assert lib.ksmm_cu_cache_append(ctypes.byref(a), None) == _lib.KSMM_ERR_BAD_ARGUMENT and text in lib.ksmm_cu_last_error()
    for kw, text in ((dict(q=None), b"null"), (dict(out=None), b"null"), (dict(window=-1), b"window"), (dict(max_new=-1), b"max_new")):
        _, t = descs(**kw)
        assert lib.ksmm_cu_cache_attention(ctypes.byref(t), None, 0, None) == _lib.KSMM_ERR_BAD_ARGUMENT
        assert text in lib.ksmm_cu_last_error()
    assert lib.ksmm_cu_cache_append(None, None) == _lib.KSMM_ERR_BAD_ARGUMENT
    assert lib.ksmm_cu_cache_attention(None, None, 0, None) == _lib.KSMM_ERR_BAD_ARGUMENT
    _, t = descs()
    assert lib.ksmm_cu_cache_attention_workspace_bytes(ctypes.byref(t)) == 0  # (a table too short for anything to be split)
    _, t = descs(table_width=4096)
    need = lib.ksmm_cu_cache_attention_workspace_bytes(ctypes.byref(t))
    assert need > 0
    for ws, size in ((None, need), (t.q, need - 1), (t.q + 16, need)):
        assert lib.ksmm_cu_cache_attention(ctypes.byref(t), ws, size, None) == _lib.KSMM_ERR_WORKSPACE
    a, t = descs(tokens=0, sequences=0)
    assert lib.ksmm_cu_cache_append(ctypes.byref(a), None) == _lib.KSMM_OK
    assert lib.ksmm_cu_cache_attention(ctypes.byref(t), None, 0, None) == _lib.KSMM_OK


def test_attention_layer_arguments():
    q, o = [(6, 64, 64, 1), (1, 192, 192, 2)], [(6, 64, 64, 1), (1, 192, 192, 2)]
    kw = dict(device="meta")
    for args, more, text in (((q, o, 5), {}, "heads"), ((q, o, 0), {}, "positive"), ((q, o, 6), dict(window=0), "positive"),
                             ((q, o, 6), dict(kv_patterns=[(6, 64, 64, 1), (1, 80, 192, 2)]), "no part"),
                             ((q, o, 6), dict(kv_patterns=[(6, 64, 64, 1), (1, 128, 192, 2)]), "no part"),
                             ((q, o, 6), dict(rotary_dim=33), "rotary_dim"), ((q, o, 6), dict(rotary_dim=66), "rotary_dim"),
                             ((q, [(1, 64, 64, 4)], 6), {}, "output layer")):
        with pytest.raises(ValueError, match=text):
            kb.KSAttention(*args, **more, **kw)
    with pytest.raises(TypeError):
        kb.KSAttention(q, o, 6, dtype=torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError):
        kb.KSAttention(q, o, 6, algo="dense")
