"""The feed-forward block's own operators as measurable cases.

A case is one of two operators, forward or as a training step:

* ``gated``: ``act(gate(x)) * up(x)`` with two Kronecker-sparse layers of the same patterns on one input
  (``KSGatedLinear``), the first half of a gated feed-forward block;
* ``norm``:  the passage from one block to the next (``residual_norm``): the block's output ``y``, normalised
  and gated, joins the residual stream ``x``, and the sum is normalised and modulated for the next block:
  ``z = alpha x + gate * post(y)``, ``h = pre(z) * (1 + scale) + shift``.

``train`` cases return the gradients of everything that learns beside the results.  Where ``own`` is false the
operators are elementary torch operations in 32 bits, rounded once at the end.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"fp32": 4, "fp16": 2, "bf16": 2}

SMALL = "6,64,64,1 1,512,192,2"                     # 384 -> 1024
BASE = "4,192,192,1 1,512,192,4"                    # 768 -> 2048
CHAIN3 = "1,64,64,16 4,64,64,4 16,176,64,1"         # 1024 -> 2816, butterfly-like
ONE = "1,512,192,4"                                 # 768 -> 2048 in one factor
EPS = 1e-5


def _gated(name, patterns, dtype, bs_last, out_last, batch, act="silu", train=False):
    return {"name": name, "op": "gated", "patterns": patterns, "dtype": dtype, "bs_last": bs_last,
            "out_last": out_last, "batch": batch, "act": act, "train": train}


def _norm(name, dtype, samples, tokens, channels, bs_last=False, pre="layer", post="none", residual=True,
          modulated=True, train=False):
    return {"name": name, "op": "norm", "dtype": dtype, "samples": samples, "tokens": tokens, "channels": channels,
            "bs_last": bs_last, "pre": pre, "post": post, "residual": residual, "modulated": modulated, "train": train}


def listed():
    return [
        # a handful of rows answered online: launches and host work are all there is
        _gated("gated_online_fp16", SMALL, "fp16", False, False, 16),
        # one image of 196 patches and a class token; the wide activations stay batch-last
        _gated("gated_image_bf16", BASE, "bf16", False, True, 197),
        # the batch of the benchmark, 128 images of 196 tokens
        _gated("gated_batch_bf16", BASE, "bf16", False, True, 25088),
        # a batch-last network on 33 images of 197 tokens: rows that are a multiple of nothing
        _gated("gated_ragged_fp16", SMALL, "fp16", True, True, 6501, act="gelu"),
        # inference in fp32 with a three-factor butterfly-like chain
        _gated("gated_chain3_fp32", CHAIN3, "fp32", False, False, 4096),
        # a training step, 64 images
        _gated("gated_train_bf16", BASE, "bf16", False, True, 12544, train=True),
        # a training step in fp32, 32 images, batch-last
        _gated("gated_train_fp32", SMALL, "fp32", True, True, 6272, train=True),
        # the norm before a block for the same handful of rows
        _norm("norm_online_fp16", "fp16", 1, 16, 384, residual=False, modulated=False),
        # between two blocks conditioned on each image, at the batch of the benchmark
        _norm("norm_images_bf16", "bf16", 128, 196, 768),
        # the same without conditioning in a batch-last network on a ragged batch
        _norm("norm_ragged_fp16", "fp16", 1, 6501, 768, bs_last=True, modulated=False),
        # a training step between conditioned blocks with a norm on both sides, 64 images with class tokens
        _norm("norm_train_bf16", "bf16", 64, 197, 768, pre="rms", post="rms", train=True),
        # a wide model over long sequences
        _norm("norm_wide_bf16", "bf16", 4, 8192, 4096, pre="rms", post="none", modulated=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        patterns = rng.choice((SMALL, BASE, CHAIN3, ONE))
        dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
        train = rng.random() < 0.4
        most = {"fp16": 25088, "bf16": 25088, "fp32": 4096}[dtype] // (2 if train else 1)
        if patterns == CHAIN3:
            most //= 2
        bs_last, out_last = rng.choice(((False, False), (False, True), (True, True), (True, False)))
        case = _gated("", patterns, dtype, bs_last, out_last, _log(rng, 1, most),
                      act=rng.choice(("silu", "silu", "gelu", "sigmoid" if train else "relu")), train=train)
    else:
        dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
        train = rng.random() < 0.4
        channels = _log(rng, 48, 8192)
        if rng.random() < 0.6:
            channels = max(channels // 64 * 64, 64)
        most = (1 << 25) // (ESIZE[dtype] * (2 if train else 1) // 2)
        samples = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(2, min(8192, most // (channels * samples))))
        case = _norm("", dtype, samples, tokens, channels, bs_last=rng.random() < 0.35, pre=rng.choice(("layer", "rms")),
                     post=rng.choice(("none", "layer", "rms")), residual=rng.random() < 0.75,
                     modulated=rng.random() < 0.6, train=train)
        if not case["residual"]:
            case["post"] = "none"
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _patterns(case):
    return [tuple(int(v) for v in p.split(",")) for p in case["patterns"].split()]


def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _gated_sizes(case):
    pats = _patterns(case)
    a, _, c, d = pats[0]
    la, lb, _, ld = pats[-1]
    return pats, a * c * d, la * lb * ld


def _prepare_gated(case, gen):
    pats, n_in, n_out = _gated_sizes(case)
    dtype, batch = DTYPES[case["dtype"]], case["batch"]
    # what a LayerNorm hands on, and the layer's own initialisation
    x = _randn(gen, *((n_in, batch) if case["bs_last"] else (batch, n_in))).to(dtype)
    factors = [((torch.rand(2 * a * d * c, b, device="cuda", generator=gen) * 2 - 1) / math.sqrt(c)).to(dtype)
               for a, b, c, d in pats]
    bias = ((torch.rand(2 * n_out, device="cuda", generator=gen) * 2 - 1) / math.sqrt(n_in)).to(dtype)
    state = {"case": case, "x": x, "factors": factors, "bias": bias}
    if case["train"]:
        state["grad"] = _randn(gen, *((n_out, batch) if case["out_last"] else (batch, n_out))).to(dtype)
    if own:
        import ksmm_b200 as kb

        layer = kb.KSGatedLinear(pats, bias=True, algo="kernel", dtype=dtype, bs_last=case["bs_last"], device="cuda",
                                 activation=case["act"], out_bs_last=case["out_last"], requires_grad=case["train"])
        with torch.no_grad():
            for p, f in zip(layer.factors, factors):
                p.copy_(f)
            layer.bias.copy_(bias.reshape(layer.bias.shape))
        state["layer"] = layer
        if case["train"]:
            state["leaf"] = x.clone().requires_grad_(True)
    return state


def _prepare_norm(case, gen):
    S, T, C = case["samples"], case["tokens"], case["channels"]
    dtype, rows = DTYPES[case["dtype"]], S * T
    shape = (C, rows) if case["bs_last"] else (S, T, C)
    # a residual stream: a few channels stand out, every token has an offset of its own
    spread = 1.0 + 4.0 * (torch.rand(C, device="cuda", generator=gen) > 0.98)
    spread = spread.reshape(-1, 1) if case["bs_last"] else spread
    x = (_randn(gen, *shape) * spread + 0.1).to(dtype)
    state = {"case": case, "x": x, "weight": (1 + 0.1 * _randn(gen, C)).to(dtype)}
    state["bias"] = (0.1 * _randn(gen, C)).to(dtype) if case["pre"] == "layer" else None
    if case["residual"]:
        state["y"] = _randn(gen, *shape).to(dtype)
    if case["modulated"]:
        # what the conditioning network returns: one row for each image, cut into its parts
        chunks = (0.3 * _randn(gen, S, 3 * C)).to(dtype)
        state["scale"], state["shift"] = chunks[:, :C], chunks[:, C:2 * C]
        if case["residual"]:
            state["gate"] = chunks[:, 2 * C:]
    elif case["residual"]:
        state["gate"] = (0.5 + 0.1 * _randn(gen, C)).to(dtype)    # a residual scale for each channel
    if case["post"] != "none":
        state["post_weight"] = (1 + 0.1 * _randn(gen, C)).to(dtype)
        if case["post"] == "layer":
            state["post_bias"] = (0.1 * _randn(gen, C)).to(dtype)
    state["alpha"] = 1.0
    if case["train"]:
        state["grad_h"] = _randn(gen, *shape).to(dtype)
        if case["residual"]:
            state["grad_z"] = _randn(gen, *shape).to(dtype)
    if own and case["train"]:
        state["leaves"] = {k: state[k].detach().clone().requires_grad_(True) for k in _norm_learned(state)}
    return state


NORM_INPUTS = ("x", "y", "weight", "bias", "scale", "shift", "gate", "post_weight", "post_bias")


def _norm_learned(state):
    return [k for k in NORM_INPUTS if state.get(k) is not None]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_gated(case, gen) if case["op"] == "gated" else _prepare_norm(case, gen)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_gated(state):
    layer = state["layer"]
    if not state["case"]["train"]:
        return layer(state["x"])
    h = layer(state["leaf"])
    grads = torch.autograd.grad(h, [state["leaf"], *layer.factors, layer.bias], state["grad"])
    return (h.detach(), *grads[:-1], grads[-1].reshape(-1))


def _own_norm(state):
    import ksmm_b200 as kb

    case = state["case"]
    src = state["leaves"] if case["train"] else state
    kw = {k: src[k] for k in NORM_INPUTS[2:] if src.get(k) is not None}
    out = kb.residual_norm(src["x"], src.get("y"), norm=case["pre"], post_norm=None if case["post"] == "none" else case["post"],
                           alpha=state["alpha"], eps=EPS, bs_last=case["bs_last"], **kw)
    if not case["train"]:
        return out
    names = _norm_learned(state)
    if case["residual"]:
        grads = torch.autograd.grad(out, [src[k] for k in names], (state["grad_z"], state["grad_h"]))
        return (out[0].detach(), out[1].detach(), *grads)
    return (out.detach(), *torch.autograd.grad(out, [src[k] for k in names], state["grad_h"]))


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _factor(x, w, p):
    """(batch, a*c*d) times one kernel-format factor: a*d products of (batch, c) and (c, b)."""
    a, b, c, d = p
    n = x.shape[0]
    blocks = x.reshape(n, a, c, d).permute(1, 3, 0, 2).reshape(a * d, n, c)
    out = torch.matmul(blocks, w.reshape(a * d, c, b))
    return out.reshape(a, d, n, b).permute(2, 0, 3, 1).reshape(n, a * b * d)


def _factor_grads(x, w, g, p):
    a, b, c, d = p
    n = x.shape[0]
    xb = x.reshape(n, a, c, d).permute(1, 3, 0, 2).reshape(a * d, n, c)
    gb = g.reshape(n, a, b, d).permute(1, 3, 0, 2).reshape(a * d, n, b)
    dw = torch.matmul(xb.transpose(1, 2), gb).reshape(a * d * c, b)
    dx = torch.matmul(gb, w.reshape(a * d, c, b).transpose(1, 2))
    return dx.reshape(a, d, n, c).permute(2, 0, 3, 1).reshape(n, a * c * d), dw


def _erf(x):
    return torch.erf(x * math.sqrt(0.5))


def _activation(g, act):
    """The activation and its derivative."""
    if act == "relu":
        pos = (g > 0).to(g.dtype)
        return g * pos, pos
    if act == "gelu":
        cdf = 0.5 * (1 + _erf(g))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return s, s * (1 - s)
    return g * s, s * (1 + g * (1 - s))


def _plain_gated(state):
    case = state["case"]
    pats, _, n_out = _gated_sizes(case)
    dtype = DTYPES[case["dtype"]]
    x = state["x"].float()
    x = x.t() if case["bs_last"] else x
    kept, outs = [], []
    for q in range(2):
        y, inputs = x, []
        for p, w in zip(pats, state["factors"]):
            inputs.append(y)
            y = _factor(y, w.float().chunk(2)[q], p)
        kept.append(inputs)
        outs.append(y + state["bias"].float()[q * n_out:(q + 1) * n_out])
    g, u = outs
    value, slope = _activation(g, case["act"])

    def laid(t, last):
        return (t.t() if last else t).contiguous().to(dtype)

    h = laid(value * u, case["out_last"])
    if not case["train"]:
        return h
    dh = state["grad"].float()
    dh = dh.t() if case["out_last"] else dh
    dx, dws, dbs = 0, [[], []], []
    for q, d in enumerate((dh * u * slope, dh * value)):
        dbs.append(d.sum(0))
        for f in range(len(pats) - 1, -1, -1):
            d, dw = _factor_grads(kept[q][f], state["factors"][f].float().chunk(2)[q], d, pats[f])
            dws[q].insert(0, dw)
        dx = dx + d
    return (h, laid(dx, case["bs_last"]), *[torch.cat(pair).to(dtype) for pair in zip(*dws)], torch.cat(dbs).to(dtype))


def _rows(t, case):
    """(samples, tokens, channels) of an activation, in 32 bits."""
    t = t.float()
    t = t.t() if case["bs_last"] else t
    return t.reshape(case["samples"], case["tokens"], case["channels"])


def _per_sample(t, case):
    return t.float().reshape(-1, 1, case["channels"])


def _normed(t, kind):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
    return t * r, r


def _normed_grad(n, r, g, kind):
    g = g - n * (g * n).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == "layer" else 0)
    return g * r


def _plain_norm(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    get = lambda k: None if state.get(k) is None else _per_sample(state[k], case)

    def laid(t):
        t = t.to(dtype)
        return t.reshape(-1, case["channels"]).t().contiguous() if case["bs_last"] else t

    z = _rows(state["x"], case)
    if case["residual"]:
        y = _rows(state["y"], case)
        if case["post"] != "none":
            yn, yr = _normed(y, case["post"])
            py = yn * get("post_weight") + (get("post_bias") if case["post"] == "layer" else 0)
        else:
            yn = py = y
        z = state["alpha"] * z + get("gate") * py
    n, r = _normed(z, case["pre"])
    m = n * get("weight") + (get("bias") if case["pre"] == "layer" else 0)
    h = m * (1 + get("scale")) + get("shift") if case["modulated"] else m
    results = (laid(z), laid(h)) if case["residual"] else laid(h)
    if not case["train"]:
        return results
    dh = _rows(state["grad_h"], case)
    grads = {}
    dm = dh
    if case["modulated"]:
        grads["scale"], grads["shift"] = (dh * m).sum(1), dh.sum(1)
        dm = dh * (1 + get("scale"))
    grads["weight"], grads["bias"] = (dm * n).sum((0, 1)), dm.sum((0, 1))
    dz = _normed_grad(n, r, dm * get("weight"), case["pre"])
    if case["residual"]:
        dz = dz + _rows(state["grad_z"], case)
        dgate = (dz * py).sum(1)
        grads["gate"] = dgate if case["modulated"] else dgate.sum(0)
        dp = dz * get("gate")
        if case["post"] != "none":
            grads["post_weight"], grads["post_bias"] = (dp * yn).sum((0, 1)), dp.sum((0, 1))
            dp = _normed_grad(yn, yr, dp * get("post_weight"), case["post"])
        grads["y"] = laid(dp)
    grads["x"] = laid(state["alpha"] * dz)
    out = results if case["residual"] else (results,)
    return (*out, *[grads[k].to(dtype) for k in _norm_learned(state)])


def run(state):
    if state["case"]["op"] == "gated":
        return _own_gated(state) if own else _plain_gated(state)
    return _own_norm(state) if own else _plain_norm(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_gated(state):
    """Every factor as the tensor K[i, j, k, l] of its definition, y[(i, j, l)] = sum_k K[i, j, k, l] x[(i, k, l)];
    gradients by differentiation of that."""
    case = state["case"]
    pats, _, n_out = _gated_sizes(case)
    train = case["train"]
    leaf = lambda t: t.double().requires_grad_(train)
    x, bias, factors = leaf(state["x"]), leaf(state["bias"]), [leaf(f) for f in state["factors"]]
    halves = []
    for q in range(2):
        y = x if case["bs_last"] else x.t()
        for (a, b, c, d), w in zip(pats, factors):
            k = w.reshape(2, a, d, c, b)[q].permute(0, 3, 2, 1)
            y = torch.einsum("ijkl,ikln->ijln", k, y.reshape(a, c, d, -1)).reshape(a * b * d, -1)
        halves.append(y + bias.reshape(2, n_out, 1)[q])
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu,
           "sigmoid": torch.sigmoid}[case["act"]]
    h = act(halves[0]) * halves[1]
    h = h if case["out_last"] else h.t()
    if not train:
        return h.contiguous()
    grads = torch.autograd.grad(h, [x, *factors, bias], state["grad"].double())
    return (h.detach().contiguous(), *grads)


def _exact_norm(state):
    case = state["case"]
    C, train = case["channels"], case["train"]
    t = {k: state[k].double().requires_grad_(train) for k in _norm_learned(state)}
    shaped = lambda v: (v.t() if case["bs_last"] else v).reshape(case["samples"], case["tokens"], C)

    def norm(v, kind, weight, bias):
        if kind == "layer":
            return torch.nn.functional.layer_norm(v, (C,), weight, bias, EPS)
        return torch.nn.functional.rms_norm(v, (C,), weight, EPS)

    z = shaped(t["x"])
    if case["residual"]:
        y = shaped(t["y"])
        if case["post"] != "none":
            y = norm(y, case["post"], t["post_weight"], t.get("post_bias"))
        z = state["alpha"] * z + t["gate"].reshape(-1, 1, C) * y
    h = norm(z, case["pre"], t["weight"], t.get("bias"))
    if case["modulated"]:
        h = h * (1 + t["scale"][:, None]) + t["shift"][:, None]
    back = lambda v: v.reshape(-1, C).t() if case["bs_last"] else v
    outs = (back(z), back(h)) if case["residual"] else (back(h),)
    done = tuple(v.detach().contiguous() for v in outs)
    if not train:
        return done if case["residual"] else done[0]
    seeds = [state[k].double() for k in ("grad_z", "grad_h") if state.get(k) is not None]
    return (*done, *torch.autograd.grad(outs, list(t.values()), seeds))


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_gated(state) if case["op"] == "gated" else _exact_norm(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    es = ESIZE[case["dtype"]]
    if case["op"] == "gated":
        pats, n_in, n_out = _gated_sizes(case)
        weights = sum(2 * a * b * c * d for a, b, c, d in pats) + 2 * n_out
        products = 2.0 * case["batch"] * sum(2 * a * b * c * d for a, b, c, d in pats)
        values = case["batch"] * (n_in + n_out)
        if case["train"]:     # also: the gradient of the output read, those of the input and of the weights written
            return {"bytes": es * (2 * values + 2 * weights), "flops": 3 * products}
        return {"bytes": es * (values + weights), "flops": products}
    S, C = case["samples"], case["channels"]
    values = S * case["tokens"] * C
    tensors = 4 if case["residual"] else 2              # x, y, z, h
    params = C * (1 + (case["pre"] == "layer") + (case["post"] != "none") + (case["post"] == "layer"))
    if case["modulated"]:
        params += S * C * (3 if case["residual"] else 2)
    elif case["residual"]:
        params += C
    flops = values * (8 + (3 if case["residual"] else 0) + (6 if case["post"] != "none" else 0))
    if case["train"]:         # the gradients of the results read, those of the inputs written
        return {"bytes": es * (2 * tensors * values + 2 * params), "flops": 3.0 * flops}
    return {"bytes": es * (tensors * values + params), "flops": float(flops)}
