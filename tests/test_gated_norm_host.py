"""Arguments that KSGatedLinear, gated_chain_forward and residual_norm refuse, and their C entry points; no GPU."""
import ctypes

import pytest
import torch

import ksmm_b200 as kb
from ksmm_b200 import _lib


def test_layer_arguments():
    pats = [(6, 64, 64, 1), (1, 512, 192, 2)]
    with pytest.raises(ValueError, match="activation"):
        kb.KSGatedLinear(pats, activation="tanh")
    with pytest.raises(ValueError, match="feeds"):
        kb.KSGatedLinear([(6, 64, 64, 1), (1, 512, 192, 4)])
    with pytest.raises(ValueError, match="factors"):
        kb.KSGatedLinear([])
    with pytest.raises(ValueError, match="factors"):
        kb.KSGatedLinear([(1, 4, 4, 1)] * 17)
    with pytest.raises(TypeError):
        kb.KSGatedLinear(pats, dtype=torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError):
        kb.KSGatedLinear(pats, algo="dense")
    with pytest.raises(Exception, match="cuda"):
        kb.KSGatedLinear(pats, device="cpu")


def test_calls_on_host_tensors():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        kb.residual_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        kb.gated_chain_forward(x, [torch.zeros(16, 8)], [(1, 8, 8, 1)], False)
    with pytest.raises(ValueError, match="norm"):
        kb.residual_norm(x, norm="batch")
    with pytest.raises(ValueError, match="activation"):
        kb.gated_chain_forward(x, [torch.zeros(16, 8)], [(1, 8, 8, 1)], False, activation="swish")


def test_module_arguments():
    with pytest.raises(ValueError):
        kb.ResidualNorm(8, norm="batch", device="cpu")
    with pytest.raises(ValueError):
        kb.ResidualNorm(0, device="cpu")
    m = kb.ResidualNorm(8, norm="rms", post_norm="layer", residual_scale=0.1, device="cpu")
    assert set(m.state_dict()) == {"weight", "post_weight", "post_bias", "gate"}
    with pytest.raises(ValueError, match="gate"):
        m(torch.zeros(2, 8), gate=torch.zeros(8))


def norm_desc(**kw):
    buf = ctypes.create_string_buffer(256)
    p = ctypes.addressof(buf)
    base = dict(x=p, h=p, rows=4, samples=1, channels=8, norm=1, post_norm=0, bs_last=0, dtype=0, param_dtype=0, alpha=1.0, eps=1e-5)
    d = _lib.NormDesc(**{**base, **kw})
    d._keep = buf
    return d


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), _lib.KSMM_ERR_UNSUPPORTED), (dict(dtype=9), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(dtype=1, param_dtype=2), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(norm=3), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(norm=0), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(post_norm=1), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(bs_last=2), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(rows=-1), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(channels=0), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(channels=8193), _lib.KSMM_ERR_UNSUPPORTED),
    (dict(samples=3), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(samples=0), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(scale_stride=-8), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(eps=-1.0), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(eps=float("nan")), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(x=None), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(h=None), _lib.KSMM_ERR_BAD_ARGUMENT),
])
def test_norm_entry(change, status):
    lib = _lib.load()
    assert lib.ksmm_cu_norm_forward(ctypes.byref(norm_desc(**change)), None, 0, None) == status
    assert lib.ksmm_cu_last_error()


def test_norm_entries_of_nothing():
    lib = _lib.load()
    before = lib.ksmm_cu_launch_count()
    assert lib.ksmm_cu_norm_forward(None, None, 0, None) == _lib.KSMM_ERR_BAD_ARGUMENT
    assert lib.ksmm_cu_norm_forward(ctypes.byref(norm_desc(rows=0, x=None, h=None)), None, 0, None) == _lib.KSMM_OK
    wide = norm_desc(bs_last=1, channels=2000)
    assert lib.ksmm_cu_norm_forward_workspace_bytes(ctypes.byref(wide)) >= 2 * 2000 * 4 * 4
    assert lib.ksmm_cu_norm_forward(ctypes.byref(wide), None, 0, None) == _lib.KSMM_ERR_WORKSPACE
    d = norm_desc()
    assert lib.ksmm_cu_norm_forward_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.ksmm_cu_norm_backward(ctypes.byref(d), None, 0, None) == _lib.KSMM_ERR_BAD_ARGUMENT   # no statistics
    d = norm_desc(grad_h=d.x, stats=(d.x + 15) // 16 * 16, grad_weight=d.x)
    need = lib.ksmm_cu_norm_backward_workspace_bytes(ctypes.byref(d))
    assert need >= 4 * 8 * 4
    assert lib.ksmm_cu_norm_backward(ctypes.byref(d), None, 0, None) == _lib.KSMM_ERR_WORKSPACE
    d = norm_desc(grad_z=d.x, stats=(d.x + 15) // 16 * 16)
    assert lib.ksmm_cu_norm_backward(ctypes.byref(d), None, 0, None) == _lib.KSMM_ERR_BAD_ARGUMENT   # no y
    assert lib.ksmm_cu_launch_count() == before


def gated_desc(patterns=((1, 8, 8, 1),), **kw):
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    n = len(patterns)
    base = dict(input=p, values=(ctypes.c_void_p * n)(*[p] * n), output=p, batch=4, nfactors=n,
                patterns=_lib.int32_array([v for q in patterns for v in q]), dtype=1, bs_last=0, out_layout=0, activation=3)
    d = _lib.GatedDesc(**{**base, **kw})
    d._keep = buf
    return d


@pytest.mark.parametrize("change,status", [
    (dict(activation=5), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(activation=-1), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(dtype=3), _lib.KSMM_ERR_UNSUPPORTED), (dict(dtype=7), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(out_layout=3), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(bs_last=2), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(batch=-1), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(input=None), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(output=None), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(values=(ctypes.c_void_p * 1)(None)), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(patterns=((1, 8, 8, 1), (1, 4, 4, 1))), _lib.KSMM_ERR_BAD_ARGUMENT), (dict(patterns=((0, 8, 8, 1),)), _lib.KSMM_ERR_BAD_ARGUMENT),
    (dict(patterns=((1, 8, 8, 1),) * 17), _lib.KSMM_ERR_UNSUPPORTED), ({}, _lib.KSMM_ERR_WORKSPACE),
])
def test_gated_entry(change, status):
    lib = _lib.load()
    change = dict(change)
    d = gated_desc(change.pop("patterns", ((1, 8, 8, 1),)), **change)
    before = lib.ksmm_cu_launch_count()
    assert lib.ksmm_cu_gated_forward(ctypes.byref(d), None) == status
    assert lib.ksmm_cu_last_error() and lib.ksmm_cu_launch_count() == before


def test_gated_training_entries():
    lib = _lib.load()
    pats = ((6, 64, 64, 1), (1, 512, 192, 2))
    sizes = (ctypes.c_size_t * 3)()
    at = [ctypes.cast(ctypes.byref(sizes, 8 * q), ctypes.POINTER(ctypes.c_size_t)) for q in range(3)]
    pat = _lib.int32_array([v for q in pats for v in q])
    assert lib.ksmm_cu_gated_train_bytes(2, pat, 100, 1, 0, 1, *at) == _lib.KSMM_OK
    assert sizes[0] >= 2 * 2 * 100 * (384 + 1024) and sizes[2] >= 2 * 2 * 100 * 1024
    assert lib.ksmm_cu_gated_train_bytes(2, pat, 0, 1, 0, 1, *at) == _lib.KSMM_OK and list(sizes) == [0, 0, 0]
    assert lib.ksmm_cu_gated_train_bytes(2, pat, 100, 1, 0, 2, *at) == _lib.KSMM_ERR_BAD_ARGUMENT
    assert lib.ksmm_cu_gated_workspace_bytes(2, pat, 100, 1, 0, 1) > 0
    assert lib.ksmm_cu_gated_workspace_bytes(2, pat, 100, 3, 0, 1) == 0
    d = gated_desc()
    p = d.input
    grads = (ctypes.c_void_p * 1)(None)
    assert lib.ksmm_cu_gated_backward(ctypes.byref(d), p, None, grads, None, None) == _lib.KSMM_ERR_BAD_ARGUMENT  # nothing kept
    layouts = (ctypes.c_int32 * 1)(7)
    d = gated_desc(saved=p, saved_bytes=4096, layouts=layouts)
    assert lib.ksmm_cu_gated_backward(ctypes.byref(d), d.input, None, grads, None, None) == _lib.KSMM_ERR_BAD_ARGUMENT
    layouts[0] = 0
    assert lib.ksmm_cu_gated_backward(ctypes.byref(d), d.input, None, grads, None, None) == _lib.KSMM_ERR_WORKSPACE
    d = gated_desc(saved=p, saved_bytes=1, layouts=layouts)
    assert lib.ksmm_cu_gated_forward(ctypes.byref(d), None) == _lib.KSMM_ERR_WORKSPACE
    d = gated_desc(saved=p, saved_bytes=4096)
    assert lib.ksmm_cu_gated_forward(ctypes.byref(d), None) == _lib.KSMM_ERR_BAD_ARGUMENT   # nowhere for the layouts
