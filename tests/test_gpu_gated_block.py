"""The gated layer and the norms together, as a block of a network uses them, against the same block in 64 bits;
calls under a captured graph, on another stream, with part of the gradients; what is refused; what stays untouched.

Tolerances of the block, relative 2-norms with u = eps / 2 of the type: z and n are rounded once each (2 u), the
gated layer adds (3 n + 1) u to three times what it is given (n = 2 factors: 7 u + 6 u), the down projection rounds
per factor (2 u) and the sum once, so 18 u for its share; doubled for short vectors, 36 u.  Gradients pass the
same steps twice: 72 u.
"""
import pytest
import torch

import ksmm_b200 as kb
from ksmm_b200.ksvit import KSGatedFeedForward, KSViTB

pytestmark = pytest.mark.gpu


def dense(factor, pattern):
    a, b, c, d = pattern
    w = factor.reshape(a, d, c, b).permute(0, 3, 2, 1)
    rows = torch.diag_embed(w).permute(0, 1, 3, 2, 4).reshape(a, b * d, c * d)
    return torch.block_diag(*torch.unbind(rows, dim=0))


def chain(x, factors, patterns):
    for f, p in zip(factors, patterns):
        x = x @ dense(f, p).t()
    return x


def block_64(x, a, p, ff):
    z = x + a
    n = torch.nn.functional.layer_norm(z, (z.shape[-1],), p["norm.weight"], p["norm.bias"], ff.norm.eps)
    flat = n.reshape(-1, n.shape[-1])
    halves = []
    for q in range(2):
        fs = [p[f"gate_up.factors.{i}"].chunk(2)[q] for i in range(2)]
        halves.append(chain(flat, fs, ff.gate_up.patterns) + p["gate_up.bias"].chunk(2)[q])
    h = torch.nn.functional.silu(halves[0]) * halves[1]
    y = chain(h, [p[f"down.factors.{i}"] for i in range(2)], ff.down.patterns) + p["down.bias"].reshape(1, -1)
    return z + y.view(z.shape)


def err(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 5), (3, 197)])
def test_block(dtype, shape):
    torch.manual_seed(0)
    ff = KSGatedFeedForward(dtype, "cuda", requires_grad=True)
    x, a = (torch.randn(*shape, 768, device="cuda").to(dtype) for _ in range(2))
    u = torch.finfo(dtype).eps / 2
    p = {k: v.detach().double().requires_grad_(True) for k, v in ff.named_parameters()}
    xe, ae = (t.double().requires_grad_(True) for t in (x, a))
    want = block_64(xe, ae, p, ff)
    with torch.no_grad():
        assert err(ff(x, a), want) <= 36 * u
    xl, al = (t.clone().requires_grad_(True) for t in (x, a))
    got = ff(xl, al)
    assert err(got, want) <= 36 * u
    seed = torch.randn_like(x)
    grads = torch.autograd.grad(got, [xl, al, *ff.parameters()], seed)
    ref = torch.autograd.grad(want, [xe, ae, *p.values()], seed.double())
    for name, g, r in zip(["x", "a", *p], grads, ref):
        assert g.shape == r.shape or g.numel() == r.numel()
        assert err(g.reshape(r.shape), r) <= 72 * u, name


def test_network_of_gated_blocks():
    torch.manual_seed(1)
    net = KSViTB(dtype=torch.bfloat16, depth=2, gated_mlp=True)
    img = torch.randn(2, 3, 224, 224, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        out = net(img)
    assert out.shape == (2, 1000) and torch.isfinite(out.float()).all()


def gated(dtype=torch.bfloat16, **kw):
    torch.manual_seed(2)
    return kb.KSGatedLinear([(6, 64, 64, 1), (1, 512, 192, 2)], dtype=dtype, **kw)


@pytest.mark.parametrize("train", [False, True])
def test_captured_and_replayed(train):
    layer = gated(requires_grad=train, out_bs_last=True)
    norm = kb.ResidualNorm(384, dtype=torch.bfloat16, post_norm="rms", residual_scale=0.5, requires_grad=train)
    x, y = (torch.randn(2560, 384, device="cuda").bfloat16() for _ in range(2))
    seed = torch.randn(1024, 2560, device="cuda").bfloat16()

    def step(x, y):
        z, n = norm(x, y)
        h = layer(n)
        if not train:
            return z, h
        return (h.detach(), *torch.autograd.grad(h, [*layer.parameters(), norm.weight, norm.gate], seed))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(x, y)
    for s in range(2):
        torch.manual_seed(10 + s)
        x.copy_(torch.randn(2560, 384, device="cuda"))
        y.copy_(torch.randn(2560, 384, device="cuda"))
        graph.replay()
        fresh = step(x, y)
        for a, b in zip(kept, fresh):
            assert torch.equal(a, b)     # (sums have a fixed order)


def test_two_streams_at_once():
    layer = gated()
    xs = [torch.randn(3001, 384, device="cuda").bfloat16() for _ in range(2)]
    want = [(layer(x), kb.residual_norm(x, x, gate=layer.factors[0][:1, :1].expand(1, 384).reshape(-1))) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = layer(xs[i]), kb.residual_norm(xs[i], xs[i], gate=layer.factors[0][:1, :1].expand(1, 384).reshape(-1))
        torch.cuda.synchronize()
        for (h, (z, n)), (hw, (zw, nw)) in zip(got, want):
            assert torch.equal(h, hw) and torch.equal(z, zw) and torch.equal(n, nw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_last", [False, True])
def test_part_of_the_gradients(dtype, out_last):
    """A gradient is the same whatever else is asked for."""
    layer = gated(dtype, requires_grad=True, out_bs_last=out_last)
    x = torch.randn(300, 384, device="cuda").to(dtype).requires_grad_(True)
    params = [x, *layer.factors, layer.bias]
    h = layer(x)
    seed = torch.randn_like(h)
    full = torch.autograd.grad(h, params, seed, retain_graph=True)
    for i, p in enumerate(params):
        for q in params:
            q.requires_grad_(q is p)
        (one,) = torch.autograd.grad(layer(x), [p], seed)
        assert torch.allclose(one.float(), full[i].float(), rtol=0, atol=4 * torch.finfo(dtype).eps * full[i].abs().max().item())


@pytest.mark.parametrize("bs_last", [False, True])
def test_one_of_two_results_learns(bs_last):
    x, y, w = (torch.randn(96, 96, device="cuda", requires_grad=True) for _ in range(3))
    w = w[0]
    z, h = kb.residual_norm(x, y, weight=w, bs_last=bs_last)
    g = torch.randn_like(x)
    (gx,) = torch.autograd.grad(z, [x], g, retain_graph=True)
    assert torch.equal(gx, g)
    only_h = torch.autograd.grad(h, [x, y], g, retain_graph=True)
    both = torch.autograd.grad([z, h], [x, y], [torch.zeros_like(g), g])
    for a, b in zip(only_h, both):
        assert torch.equal(a, b)


def test_gradients_by_differences():
    """fp32: a directional derivative against central differences of the results.  With a step of 2^-7 the truncation
    is the third derivative's, about step^2 / 6 = 1e-5 of the derivative's size, and the rounding of both results,
    1e-6 each on sums of 3e5 products, divided by the step, 1e-4 of theirs: 2e-3 covers both with a margin for the
    cancellation between directions."""
    torch.manual_seed(3)
    layer = gated(torch.float32, requires_grad=True)
    x = torch.randn(300, 384, device="cuda", requires_grad=True)
    y, w, sc = torch.randn(300, 384, device="cuda", requires_grad=True), torch.randn(384, device="cuda", requires_grad=True), \
        torch.randn(3, 384, device="cuda", requires_grad=True)

    def f(x, y, w, sc):
        z, n = kb.residual_norm(x, y, norm="rms", post_norm="layer", weight=w, scale=sc, gate=w)
        return layer(n).double().pow(2).sum() + z.double().pow(3).sum() * 0.1

    args = (x, y, w, sc)
    grads = torch.autograd.grad(f(*args), args)
    step = 2.0 ** -7
    for i in range(4):
        v = torch.randn_like(args[i]) / args[i].numel() ** 0.5
        with torch.no_grad():
            plus = f(*[t + step * v if j == i else t for j, t in enumerate(args)])
            minus = f(*[t - step * v if j == i else t for j, t in enumerate(args)])
        slope = ((plus - minus) / (2 * step)).item()
        assert abs(slope - (grads[i].double() * v.double()).sum().item()) <= 2e-3 * grads[i].double().norm().item() * v.double().norm().item()


def test_rows_of_nothing():
    layer = gated(requires_grad=True)
    x = torch.empty(0, 384, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    h = layer(x)
    assert h.shape == (0, 1024)
    gx, *gw = torch.autograd.grad(h, [x, *layer.parameters()], torch.empty_like(h))
    assert gx.shape == x.shape and all((g == 0).all() for g in gw)
    w = torch.ones(384, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    z, n = kb.residual_norm(x, x, weight=w, gate=w)
    assert z.shape == n.shape == x.shape
    assert (torch.autograd.grad([z, n], [w], [z, n])[0] == 0).all()


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("rows", [40, 2600])
def test_a_row_keeps_its_infinities_and_nans(kind, bs_last, rows):
    x = torch.randn(rows, 256, device="cuda").bfloat16()
    bad = x.clone()
    bad[3, 7], bad[11, 100], bad[12, 0] = float("nan"), float("inf"), -float("inf")
    lay = (lambda t: t.t().contiguous()) if bs_last else (lambda t: t)
    a, b = (kb.residual_norm(lay(t), norm=kind, bs_last=bs_last) for t in (x, bad))
    a, b = lay(a), lay(b)
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[[3, 11, 12]] = False
    assert torch.equal(a[others], b[others]) and not torch.isfinite(b[~others].float()).all(-1).any()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("out_last", [False, True])
@pytest.mark.parametrize("rows", [40, 2600])
def test_a_token_keeps_its_infinities_and_nans_gated(act, out_last, rows):
    layer = gated(activation=act, out_bs_last=out_last)
    x = torch.randn(rows, 384, device="cuda").bfloat16()
    bad = x.clone()
    bad[2, 5], bad[9, 300] = float("nan"), float("inf")
    lay = (lambda t: t.t().contiguous()) if out_last else (lambda t: t)
    a, b = lay(layer(x)), lay(layer(bad))
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[[2, 9]] = False
    assert torch.equal(a[others], b[others]) and torch.isnan(b[2]).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_large_values_of_the_gate(dtype):
    """A gate far on either side of 0 neither overflows nor leaves its limits."""
    pats = [(1, 64, 64, 1)]
    eye = torch.eye(64, device="cuda").reshape(1, 64, 64, 1)
    layer = kb.KSGatedLinear(pats, gate_weights=[eye], up_weights=[eye], bias=False, dtype=dtype, activation="silu")
    x = torch.zeros(4096, 64, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = -200.0, 200.0, -60.0, 60.0
    got = layer(x).double()
    want = torch.nn.functional.silu(x.double()) * x.double()
    assert (got - want).abs().max().item() <= 4 * torch.finfo(dtype).eps * 40000 and torch.isfinite(got).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out_last", [False, True])
def test_the_lowest_gates_close(act, dtype, out_last):
    """However far below 0 a gate is, nothing passes it (sigmoid(-100) = 4e-44 rounds to 0 or a subnormal number;
    the up projection multiplies that by 1)."""
    pats = [(1, 64, 64, 1)]
    eye = torch.eye(64, device="cuda").reshape(1, 64, 64, 1)
    layer = kb.KSGatedLinear(pats, gate_weights=[eye], up_weights=[eye.roll(1, 1)], bias=False, dtype=dtype, activation=act,
                             out_bs_last=out_last)
    x = torch.zeros(512, 64, device="cuda", dtype=dtype)
    for k, v in ((0, -100.0), (2, -1e4), (4, torch.finfo(dtype).min / 2)):
        x[:, k], x[:, k - 1], x[:, (k + 1) % 64] = v, 1.0, 1.0
    got = layer(x)
    got = got.t() if out_last else got
    assert got[:, [0, 2, 4]].abs().max().item() < 1e-37


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_relu_keeps_a_nan_of_the_gate(dtype):
    layer = kb.KSGatedLinear([(1, 64, 64, 1)], bias=True, dtype=dtype, activation="relu", requires_grad=True)
    with torch.no_grad():
        layer.bias[3] = float("nan")
    out = layer(torch.randn(40, 64, device="cuda").to(dtype))
    with torch.no_grad():
        plain = layer(torch.randn(40, 64, device="cuda").to(dtype))
    for o in (out, plain):
        assert torch.isnan(o[:, 3]).all() and torch.isfinite(o[:, 4:]).all()


def test_neighbours_of_outputs_stay():
    """Outputs are written inside their bounds: rows behind the last token, columns behind the last feature."""
    for batch in (45, 197, 2601):
        layer = gated(out_bs_last=True)
        x = torch.randn(batch, 384, device="cuda").bfloat16()
        room = torch.full((1024 * batch + 4096,), 7.0, device="cuda", dtype=torch.bfloat16)
        import ctypes

        from ksmm_b200 import _lib, kernel as k
        desc, (n, feats, code) = k._gated_desc(x, list(layer.factors), layer.patterns, False, True, layer.bias, "silu")
        need = _lib.load().ksmm_cu_gated_workspace_bytes(desc.nfactors, desc.patterns, n, code, 0, 1)
        ws = torch.empty(need, device="cuda", dtype=torch.uint8)
        desc.output, desc.workspace, desc.workspace_bytes = room[2048:].data_ptr(), ws.data_ptr(), need
        _lib.check(_lib.load().ksmm_cu_gated_forward(ctypes.byref(desc), k._stream_ptr(x.device)))
        assert torch.equal(room[2048:2048 + 1024 * batch].view(1024, batch), layer(x))
        assert (room[:2048] == 7).all() and (room[2048 + 1024 * batch:] == 7).all()


def shifted(t):
    """The same values at an address that is no multiple of 16 bytes."""
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = room[1:].view(t.shape)
    return out.copy_(t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bs_last,out_last", [(False, False), (False, True), (True, True), (True, False)])
def test_addresses_of_any_alignment(dtype, bs_last, out_last):
    layer = gated(dtype, bs_last=bs_last, out_bs_last=out_last, requires_grad=True)
    x = torch.randn(*((384, 200) if bs_last else (200, 384)), device="cuda").to(dtype)
    want = layer(x.requires_grad_(True))
    seed = torch.randn_like(want)
    ref = torch.autograd.grad(want, [x, *layer.factors, layer.bias], seed)
    xs = shifted(x.detach()).requires_grad_(True)
    fs = [shifted(f.detach()).requires_grad_(True) for f in layer.factors]
    b = shifted(layer.bias.detach().reshape(-1)).requires_grad_(True)
    got = kb.kernel.gated_layer(xs, fs, layer.patterns, bs_last, b, "silu", out_last)
    # (another kernel may run: three roundings per factor on either side)
    tol = 12 * (2e-6 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    assert err(got, want.double()) <= tol
    for a, r in zip(torch.autograd.grad(got, [xs, *fs, b], shifted(seed)), ref):
        assert err(a, r.double().reshape(a.shape)) <= 2 * tol
    y = torch.randn(200, 768, device="cuda").to(dtype)
    assert torch.equal(kb.residual_norm(shifted(y), y)[0], kb.residual_norm(y, y)[0])


def test_cut_and_transposed_inputs():
    x = torch.randn(6, 50, 512, device="cuda").half()
    want = kb.residual_norm(x[:, 1:, 128:].contiguous(), norm="rms")
    assert torch.equal(kb.residual_norm(x[:, 1:, 128:], norm="rms"), want)
    layer = gated(torch.float16)
    assert torch.equal(layer(x[:, 1:, 128:]), layer(x[:, 1:, 128:].contiguous()))


def test_twice_differentiated_is_refused():
    layer = gated(torch.float32, requires_grad=True)
    x = torch.randn(64, 384, device="cuda", requires_grad=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(layer(x).sum(), [x], create_graph=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(kb.residual_norm(x).sum(), [x], create_graph=True)


@pytest.mark.parametrize("rows", [64, 2560])
def test_python_and_native_bindings_agree(rows, monkeypatch):
    layer = gated(requires_grad=True)
    x = torch.randn(rows, 384, device="cuda").bfloat16().requires_grad_(True)
    w = torch.randn(384, device="cuda").bfloat16().requires_grad_(True)

    def both():
        h = layer(x)
        z, n = kb.residual_norm(x, x, weight=w, gate=w)
        with torch.no_grad():
            free = layer(x), *kb.residual_norm(x, x, weight=w, gate=w)
        return [*free, h, z, n, *torch.autograd.grad([h, z, n], [x, w, *layer.parameters()], [h, z, n])]

    native = both()
    monkeypatch.setattr(kb.kernel, "_native", None)
    monkeypatch.setattr(kb.norm, "_native", None)
    for a, b in zip(native, both()):
        assert torch.equal(a, b)
