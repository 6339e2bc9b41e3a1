"""The passage from one block of a network to the next: norms before and after a block, its gate and residual
scale, and the modulation of the next block's input, in one kernel (``ksmm_cu_norm_forward``).

The reference's models do this in separate PyTorch calls around every pair of layers
(src/ksmm_py/model/vit.py:416-431, 770-800).
"""
from __future__ import annotations

import ctypes

import torch
from torch import nn

from . import _lib
from ._lib import native as _native
from .kernel import _result, _stream_ptr, differentiable_once, dtype_code, no_tangents

_ROWS = ("weight", "bias", "post_weight", "post_bias")
_PER_SAMPLE = ("scale", "shift", "gate")
_PARAMS = _ROWS + _PER_SAMPLE


def _plan(x, y, params, norm, post_norm, bs_last):
    """Checks everything; returns the tensors as the kernel takes them and (rows, channels, samples)."""
    if norm not in _lib.NORMS or post_norm not in _lib.NORMS:
        raise ValueError(f"norm={norm!r}, post_norm={post_norm!r}: expected None, 'layer' or 'rms'")
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"norms run in float32, float16 or bfloat16, not {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x needs a dimension of channels")
    if norm is None and y is None:
        raise ValueError("without a norm there must be a second tensor y to join x")
    channels = x.shape[0] if bs_last else x.shape[-1]
    if channels == 0:
        raise ValueError("x has no channels")
    if channels >= 2 ** 31:  # (the library takes up to 8192, in a 32-bit field)
        raise ValueError(f"x has {channels} channels")
    rows = x.numel() // channels
    if y is not None:
        if not isinstance(y, torch.Tensor) or y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
            raise ValueError("y must have x's shape, type and device")
    elif post_norm is not None or any(params[k] is not None for k in ("post_weight", "post_bias", "gate")):
        raise ValueError("post_norm, post_weight, post_bias and gate apply to y, which is not given")
    if post_norm is None and (params["post_weight"] is not None or params["post_bias"] is not None):
        raise ValueError("post_weight and post_bias belong to a post_norm")
    if norm is None and any(params[k] is not None for k in ("weight", "bias", "scale", "shift")):
        raise ValueError("weight, bias, scale and shift belong to a norm")
    samples, types = 1, set()
    for k in _PARAMS:
        p = params[k]
        if p is None:
            continue
        if not isinstance(p, torch.Tensor) or p.device != x.device:
            raise ValueError(f"{k} must be a tensor on x's device")
        if p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{k} is {p.dtype}: expected {x.dtype} or float32")
        types.add(p.dtype)
        if p.dim() == 1 and p.shape[0] == channels:
            continue
        if k in _ROWS or p.dim() != 2 or p.shape[1] != channels:
            shapes = f"({channels},)" if k in _ROWS else f"({channels},) or (samples, {channels})"
            raise ValueError(f"{k} must have shape {shapes}, got {tuple(p.shape)}")
        if p.shape[0] != 1:
            if samples != 1 and p.shape[0] != samples:
                raise ValueError(f"{k} has {p.shape[0]} samples, another parameter {samples}")
            samples = p.shape[0]
    if samples == 0 or rows % samples:
        raise ValueError(f"{rows} tokens do not divide into {samples} samples")
    ptype = x.dtype if types <= {x.dtype} else torch.float32
    made = {}
    for k in _PARAMS:
        p = params[k]
        if p is not None:
            p = p if p.dtype == ptype else p.to(ptype)
            per = p.dim() == 2 and p.shape[0] > 1
            if p.stride(-1) != 1 or (per and p.stride(0) <= 0):
                p = p.contiguous()
        made[k] = p
    return x.contiguous(), None if y is None else y.contiguous(), made, (rows, channels, samples, ptype)


def _desc(x, y, z, params, sizes, kinds):
    rows, channels, samples, ptype = sizes
    norm, post_norm, alpha, eps, bs_last = kinds
    d = _lib.NormDesc(x=x.data_ptr(), rows=rows, samples=samples, channels=channels, norm=_lib.NORMS[norm],
                      post_norm=_lib.NORMS[post_norm], bs_last=int(bool(bs_last)), dtype=dtype_code(x.dtype),
                      param_dtype=dtype_code(ptype), alpha=float(alpha), eps=float(eps))
    if y is not None:
        d.y, d.z = y.data_ptr(), None if z is None else z.data_ptr()
    for k, p in params.items():
        if p is None:
            continue
        setattr(d, k, p.data_ptr())
        if k in _PER_SAMPLE and p.dim() == 2 and p.shape[0] > 1:
            setattr(d, k + "_stride", p.stride(0))
    return d


def _forward(x, y, params, sizes, kinds, keep):
    z = torch.empty_like(x) if y is not None else None
    h = torch.empty_like(x) if kinds[0] is not None else None
    stats = torch.empty(sizes[0] * 4, dtype=torch.float32, device=x.device) if keep else None
    d = _desc(x, y, z, params, sizes, kinds)
    d.h = None if h is None else h.data_ptr()
    d.stats = None if stats is None else stats.data_ptr()
    lib = _lib.load()
    size = lib.ksmm_cu_norm_forward_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    with torch.cuda.device(x.device):
        _lib.check(lib.ksmm_cu_norm_forward(ctypes.byref(d), ws.data_ptr() if size else None, size, _stream_ptr(x.device)))
    return z, h, stats


class NormFunction(torch.autograd.Function):
    """``residual_norm`` as a differentiable operation."""

    @staticmethod
    def forward(ctx, x, y, sizes, kinds, *params):
        named = dict(zip(_PARAMS, params))
        z, h, stats = _forward(x, y, named, sizes, kinds, True)
        # (what pre normalised: 16-bit calls form it again from x and y, unrounded)
        ctx.save_for_backward(z if y is not None and x.dtype == torch.float32 else x, y, stats, *params)
        ctx.plan = (sizes, kinds)
        ctx.set_materialize_grads(False)
        return (h,) if z is None else (z,) if h is None else (z, h)

    @staticmethod
    def backward(ctx, *grads):
        differentiable_once()
        x, y, stats, *params = ctx.saved_tensors
        sizes, kinds = ctx.plan
        grad_z = grads[0] if y is not None else None
        grad_h = grads[-1] if kinds[0] is not None else None
        if grad_z is None and grad_h is None:
            return (None,) * (4 + len(params))
        keep = []  # gradients laid out as the kernel reads them
        named = dict(zip(_PARAMS, params))
        d = _desc(x, y, x if x.dtype == torch.float32 else None, named, sizes, kinds)
        d.stats = stats.data_ptr()
        for k, g in (("grad_z", grad_z), ("grad_h", grad_h)):
            if g is not None:
                keep.append(g.to(x.dtype).contiguous())
                setattr(d, k, keep[-1].data_ptr())
        need = ctx.needs_input_grad
        out = [torch.empty_like(x) if need[0] else None, torch.empty_like(x) if need[1] else None, None, None]
        out += [torch.empty(p.shape, dtype=p.dtype, device=p.device) if p is not None and n else None
                for p, n in zip(params, need[4:])]
        for k, g in zip(("x", "y"), out):
            if g is not None:
                setattr(d, "grad_" + k, g.data_ptr())
        for k, g in zip(_PARAMS, out[4:]):
            if g is not None:
                setattr(d, "grad_" + k, g.data_ptr())
        lib = _lib.load()
        size = lib.ksmm_cu_norm_backward_workspace_bytes(ctypes.byref(d))
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            _lib.check(lib.ksmm_cu_norm_backward(ctypes.byref(d), ws.data_ptr(), size, _stream_ptr(x.device)))
        return tuple(out)


def residual_norm(x, y=None, *, norm="layer", post_norm=None, weight=None, bias=None, scale=None, shift=None, gate=None,
                  post_weight=None, post_bias=None, alpha=1.0, eps=1e-5, bs_last=False):
    """Joins a block's output ``y`` to the residual stream ``x`` and prepares the next block's input::

        z = alpha * x + gate * (post_norm(y) * post_weight + post_bias)        (z = x without y)
        h = (norm(z) * weight + bias) * (1 + scale) + shift

    ``norm`` and ``post_norm``: ``"layer"``, ``"rms"`` or ``None``.  Tensors are (..., channels), or
    (channels, ...) with ``bs_last``, in fp32, fp16 or bf16; parameters have that type or fp32.  ``weight``,
    ``bias``, ``post_weight`` and ``post_bias`` are (channels,); ``scale``, ``shift`` and ``gate`` are
    (channels,) or one row per sample, (samples, channels), where a sample is a run of tokens of equal length
    (rows of any stride: parts of a conditioning network's output are taken as they are).

    Returns ``(z, h)``; ``h`` alone without ``y``; ``z`` alone with ``norm=None``.  Differentiable in every
    tensor, once and in reverse mode.  ``h`` is made from the unrounded ``z``."""
    if _native is not None and isinstance(x, torch.Tensor) and norm in _lib.NORMS and post_norm in _lib.NORMS:
        # one call of the extension module; None where it is not for it (a wrong argument, parameters of two types, ...)
        out = _native.residual_norm(x, y, weight, bias, post_weight, post_bias, scale, shift, gate, _lib.NORMS[norm],
                                    _lib.NORMS[post_norm], alpha, eps, bool(bs_last))
        if out is not None:
            return _result(out)
    no_tangents(x, y, weight, bias, post_weight, post_bias, scale, shift, gate)
    params = dict(weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, scale=scale, shift=shift, gate=gate)
    x, y, params, sizes = _plan(x, y, params, norm, post_norm, bs_last)
    kinds = (norm, post_norm, float(alpha), float(eps), bool(bs_last))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, *params.values())):
        out = NormFunction.apply(x, y, sizes, kinds, *params.values())
        return out if len(out) > 1 else out[0]
    z, h, _ = _forward(x, y, params, sizes, kinds, False)
    return h if z is None else z if h is None else (z, h)


class ResidualNorm(nn.Module):
    """``residual_norm`` with its learned rows: ``weight`` and ``bias`` of ``norm``, ``post_weight`` and
    ``post_bias`` of ``post_norm`` (biases for layer norms), and, with ``residual_scale`` (its initial value), a
    ``gate`` for each channel.  ``forward(x, y=None, scale=None, shift=None, gate=None)``; a gate passed
    there replaces the learned one."""

    def __init__(self, channels, norm="layer", post_norm=None, affine=True, residual_scale=None, alpha=1.0, eps=1e-5,
                 dtype: torch.dtype = torch.float16, bs_last: bool = False, device: str = "cuda", requires_grad: bool = False):
        super().__init__()
        if norm not in _lib.NORMS or post_norm not in _lib.NORMS:
            raise ValueError(f"norm={norm!r}, post_norm={post_norm!r}: expected None, 'layer' or 'rms'")
        if channels <= 0:
            raise ValueError("a norm needs channels")
        self.channels, self.norm, self.post_norm = int(channels), norm, post_norm
        self.alpha, self.eps, self.bs_last = float(alpha), float(eps), bool(bs_last)

        def row(there, value):
            return nn.Parameter(torch.full((self.channels,), float(value), dtype=dtype, device=device),
                                requires_grad=bool(requires_grad)) if there else None

        for prefix, kind in (("", norm), ("post_", post_norm)):
            self.register_parameter(prefix + "weight", row(affine and kind is not None, 1))
            self.register_parameter(prefix + "bias", row(affine and kind == "layer", 0))
        self.register_parameter("gate", row(residual_scale is not None, residual_scale or 0))

    def forward(self, x, y=None, scale=None, shift=None, gate=None):
        kw = {}
        if y is not None:
            kw = dict(post_norm=self.post_norm, post_weight=self.post_weight, post_bias=self.post_bias,
                      gate=self.gate if gate is None else gate)
        elif gate is not None:
            raise ValueError("a gate applies to y, which is not given")
        return residual_norm(x, y, norm=self.norm, weight=self.weight, bias=self.bias, scale=scale, shift=shift,
                             alpha=self.alpha, eps=self.eps, bs_last=self.bs_last, **kw)

    def extra_repr(self):
        return "channels={}, norm={!r}, post_norm={!r}, alpha={}, eps={}, bs_last={}".format(
            self.channels, self.norm, self.post_norm, self.alpha, self.eps, self.bs_last)
