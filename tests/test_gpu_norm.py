"""residual_norm against its definition in 64 bits, forward and backward.

Tolerances (relative 2-norm over a tensor): a result rounded once to type t is off by at most u = eps(t) / 2
per element.  Before that rounding everything is fp32: a statistic is a sum of C terms in a tree of
depth <= 40 (32 terms per thread, then warps), each step u32 = 2^-24, and enters a chain of fewer than ten
operations, so 64 u32 covers it where no cancellation occurs.  The backward pass reads z rounded to t
where there is a y (u per element on z, amplified by the spread of z over its deviation, which the inputs keep
below 2) and passes two means of such values: 8 u.  Sums over tokens average these errors: the same 8 u.
"""
import pytest
import torch

import ksmm_b200 as kb

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
PARAMS = ("weight", "bias", "scale", "shift", "gate", "post_weight", "post_bias")


def unit(t):
    return torch.finfo(t).eps / 2


def bounds(dtype):
    return unit(dtype) + 64 * 2.0 ** -24, 8 * unit(dtype) + 128 * 2.0 ** -24


def normed(v, kind, weight, bias, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    return v * (1 if weight is None else weight) + (0 if bias is None else bias)


def definition(x, y, p, norm, post_norm, alpha, eps, bs_last):
    """The results in 64 bits, from (rows, channels) views."""
    C = x.shape[0] if bs_last else x.shape[-1]
    flat = lambda t: t.reshape(C, -1).t() if bs_last else t.reshape(-1, C)
    back = lambda t: (t.t() if bs_last else t).reshape(x.shape)
    rows = x.numel() // C

    def spread(t):
        return t if t is None or t.dim() == 1 else t.repeat_interleave(rows // t.shape[0], 0)

    z = flat(x)
    if y is not None:
        q = normed(flat(y), post_norm, p["post_weight"], p["post_bias"], eps)
        z = alpha * z + (1 if p["gate"] is None else spread(p["gate"])) * q
    out = [back(z)] if y is not None else []
    if norm is not None:
        h = normed(z, norm, p["weight"], p["bias"], eps)
        if p["scale"] is not None:
            h = h * (1 + spread(p["scale"]))
        if p["shift"] is not None:
            h = h + spread(p["shift"])
        out.append(back(h))
    return out


def make(dtype, shape, bs_last, samples, keys, residual, seed=0, ptype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    C = shape[0] if bs_last else shape[-1]
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = (rnd(*shape) + 0.25).to(dtype)
    y = rnd(*shape).to(dtype) if residual else None
    p = dict.fromkeys(PARAMS)
    for k in keys:
        per = k in ("scale", "shift", "gate") and samples > 1
        v = 0.3 * rnd(*((samples, C) if per else (C,)))
        p[k] = (v + (1 if k.endswith("weight") else 0)).to(ptype or dtype)
    return x, y, p


def check(dtype, shape, norm="layer", post_norm=None, bs_last=False, samples=1, keys=(), residual=True, alpha=1.0,
          train=True, ptype=None, eps=1e-5):
    x, y, p = make(dtype, shape, bs_last, samples, keys, residual, ptype=ptype)
    C = shape[0] if bs_last else shape[-1]
    t = {"x": x, "y": y, **p}
    leaves = {k: v.clone().requires_grad_(train) for k, v in t.items() if v is not None}
    out = kb.residual_norm(leaves["x"], leaves.get("y"), norm=norm, post_norm=post_norm, alpha=alpha, bs_last=bs_last, eps=eps,
                           **{k: leaves.get(k) for k in PARAMS})
    out = out if isinstance(out, tuple) else (out,)
    exact = {k: v.double().requires_grad_(train) for k, v in t.items() if v is not None}
    want = definition(exact["x"], exact.get("y"), {k: exact.get(k) for k in PARAMS}, norm, post_norm, alpha, eps, bs_last)
    assert len(out) == len(want)
    forward, backward = bounds(dtype)
    err = lambda a, b: ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()
    for a, b in zip(out, want):
        assert a.shape == x.shape and a.dtype == dtype and a.is_contiguous()
        assert err(a, b) <= forward
    if not train:
        return
    g = torch.Generator(device="cuda").manual_seed(7)
    seeds = [torch.randn(*shape, device="cuda", generator=g).to(dtype) for _ in out]
    got = torch.autograd.grad(out, list(leaves.values()), seeds)
    ref = torch.autograd.grad(want, list(exact.values()), [s.double() for s in seeds])
    single = uncancelled(t, seeds, norm, post_norm, alpha, eps, samples) if C == 1 else {}
    for k, a, b in zip(leaves, got, ref):
        assert a.shape == leaves[k].shape and a.dtype == leaves[k].dtype
        size = single[k].norm() if k in single else b.norm().clamp_min(1e-30)
        off = ((a.double() - b).norm() / size).item()
        assert off <= backward, (k, off)


def uncancelled(t, seeds, norm, post_norm, alpha, eps, samples):
    """One channel: with n = z r, the gradient r (e - n (e n)) is e r times 1 - n^2 = eps r^2, a difference that loses
    every digit, so its error is a fraction of r |e| instead: n carries the errors of z, of r and of a product, all
    below u + 4 u32, twice as much in n^2, and the difference and its product with r three roundings more: below
    4 u + 16 u32, and `backward` is 8 u + 128 u32.  What G passes on inherits that.  Returns the magnitudes
    without the difference, which take the place of the results in the tolerance."""
    v = {k: t[k].double().reshape(-1) if t.get(k) is not None else None for k in ("x", "y", *PARAMS)}
    y, r2 = v["y"], 1 / torch.sqrt(v["y"] ** 2 + eps)
    m = y * r2 if post_norm else y
    q = m * v["post_weight"] + (v["post_bias"] if v["post_bias"] is not None else 0)
    z = alpha * v["x"] + v["gate"] * q
    big = seeds[0].double().reshape(-1).abs()
    big = big + (seeds[1].double().reshape(-1) * v["weight"] * (1 + v["scale"])).abs() / torch.sqrt(z ** 2 + eps)
    return {"x": alpha * big, "y": big * (v["gate"] * v["post_weight"]).abs() * r2, "gate": (big * q.abs()).sum(),
            "post_weight": (big * (v["gate"] * m).abs()).sum(), "post_bias": (big * v["gate"].abs()).sum()}


EVERY = ("weight", "bias", "scale", "shift", "gate", "post_weight", "post_bias")


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [1, 7, 48, 96, 1303])
def test_channels(dtype, channels, bs_last):
    # (one channel: the layer norm of a single value is its bias; rms keeps the sign)
    shape = (channels, 45) if bs_last else (45, channels)
    kind = "layer" if channels > 1 else "rms"
    check(dtype, shape, norm=kind, post_norm=kind, bs_last=bs_last, keys=EVERY)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [256, 512, 768, 1024, 2048, 4096, 8192])
def test_wide_rows(dtype, channels):
    check(dtype, (9, channels), norm="rms", post_norm="layer", keys=EVERY)


@pytest.mark.parametrize("channels", [4097, 8192])
def test_widest(channels):
    check(torch.bfloat16, (5, channels), keys=("weight", "bias", "gate"))
    check(torch.bfloat16, (channels, 5), keys=("weight", "bias", "gate"), bs_last=True)


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("rows,samples", [(1, 1), (2, 2), (33, 1), (394, 2), (392, 8), (60, 60), (6501, 1)])
def test_tokens_and_samples(rows, samples, bs_last):
    check(torch.bfloat16, (384, rows) if bs_last else (rows, 384), bs_last=bs_last, samples=samples, keys=EVERY,
          norm="layer", post_norm="rms")


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("residual,norm,post_norm,keys", [
    (False, "layer", None, ()),
    (False, "rms", None, ("weight",)),
    (False, "layer", None, ("scale", "shift")),
    (True, None, None, ("gate",)),
    (True, None, "layer", ("post_weight", "post_bias")),
    (True, "rms", None, ("weight", "scale")),
    (True, "layer", "rms", ("shift", "gate", "post_weight")),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts(dtype, residual, norm, post_norm, keys, bs_last):
    check(dtype, (192, 66) if bs_last else (66, 192), norm=norm, post_norm=post_norm, bs_last=bs_last, samples=3, keys=keys,
          residual=residual, alpha=0.75 if residual else 1.0)


@pytest.mark.parametrize("bs_last", [False, True])
def test_fp32_parameters_of_16_bit_tensors(bs_last):
    check(torch.bfloat16, (200, 34) if bs_last else (34, 200), keys=EVERY, samples=2, bs_last=bs_last, norm="layer",
          post_norm="layer", ptype=torch.float32)


def test_more_dimensions():
    check(torch.float16, (4, 3, 5, 64), keys=EVERY, samples=4, post_norm="rms")
    check(torch.float16, (64, 4, 3, 5), keys=EVERY, samples=4, post_norm="rms", bs_last=True)


@pytest.mark.parametrize("dtype,channels", [(torch.bfloat16, 64), (torch.bfloat16, 768), (torch.bfloat16, 1024), (torch.float16, 384),
                                            (torch.float32, 512), (torch.float32, 96)])
@pytest.mark.parametrize("rows,samples", [(2400, 1), (2380, 7), (12544, 64), (2368, 74)])
def test_many_rows(dtype, channels, rows, samples):
    """Runs of rows through shared memory, a warp per row; also runs shorter than the rows in flight."""
    check(dtype, (rows, channels), norm="layer", post_norm="rms", samples=samples, keys=EVERY)
    check(dtype, (rows, channels), norm="rms", residual=False, keys=("weight",), train=False)


@pytest.mark.parametrize("dtype,channels", [(torch.bfloat16, 1152), (torch.bfloat16, 4096), (torch.bfloat16, 8192), (torch.float32, 2048),
                                            (torch.float32, 8192), (torch.float16, 5000)])
@pytest.mark.parametrize("rows,samples", [(601, 1), (750, 25), (608, 2)])
def test_many_wide_rows(dtype, channels, rows, samples):
    """Runs of rows through shared memory, a block per row."""
    check(dtype, (rows, channels), norm="layer", post_norm="layer", samples=samples, keys=EVERY)
    check(dtype, (rows, channels), norm="rms", residual=False, keys=("weight",), train=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,rows,samples", [(1536, 70, 2), (1537, 70, 2), (2304, 413, 7), (4800, 115, 23), (6950, 33, 1)])
def test_wide_columns(dtype, channels, rows, samples):
    """Batch-last tensors on either side of what a block keeps of a token."""
    check(dtype, (channels, rows), norm="layer", post_norm="rms", samples=samples, keys=EVERY, bs_last=True)
    check(dtype, (channels, rows), norm="rms", residual=False, keys=("weight",), bs_last=True)
    check(dtype, (channels, rows), norm=None, post_norm="layer", keys=("post_weight",), bs_last=True)
