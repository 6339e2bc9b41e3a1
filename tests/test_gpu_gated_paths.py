"""Paths of the gated layer's kernels against the definition in 64 bits.

Tolerances are those of test_gpu_gated.py (n factors, u = eps / 2 of the type, relative 2-norms): 2 (3 n + 1) u forward,
2 (5 n + 5) u backward.
"""
import pytest
import torch
import torch.nn.utils.parametrize
import torch.nn.utils.prune

import ksmm_b200 as kb
from ksmm_b200.ksvit import KSGatedFeedForward, KSViTB
from test_gpu_gated import LAYOUTS, definition, err, layer_and_input, unit

pytestmark = pytest.mark.gpu


def params_of(layer):
    return [*layer.factors, *([] if layer.bias is None else [layer.bias])]


def exact_gradients(layer, x, seed, act, out_last):
    exact = [t.detach().double().requires_grad_(True) for t in (x, *params_of(layer))]
    n = len(layer.patterns)
    want = definition(exact[0], exact[1:1 + n], exact[-1] if layer.bias is not None else None, layer.patterns, layer.bs_last,
                      out_last, act)
    return want, torch.autograd.grad(want, exact, seed.double())


@pytest.mark.parametrize("batch", [1995, 6501])
@pytest.mark.parametrize("patterns", [[(1, 512, 160, 8)], [(1, 512, 64, 8)], [(2, 96, 64, 16)]], ids=["pairs", "four_tiles", "one_tile"])
@pytest.mark.parametrize("bs_last", [False, True])
def test_kept_halves_of_many_ragged_tiles(patterns, batch, bs_last):
    """Training with batch-last outputs whose rows no tensor map addresses: every CTA walks several tiles (3 to 12
    here), each of which stores both halves through staging tiles that the product's rows use in between."""
    layer, x = layer_and_input(patterns, torch.bfloat16, bs_last, True, batch, "silu", train=True)
    leaf = x.requires_grad_(True)
    n, u = len(patterns), unit(torch.bfloat16)
    seed = torch.randn(layer.out_size, batch, device="cuda").bfloat16()
    want, ref = exact_gradients(layer, leaf, seed, "silu", True)
    first = None
    for _ in range(4):
        h = layer(leaf)
        got = torch.autograd.grad(h, [leaf, *params_of(layer)], seed)
        assert err(h, want) <= 2 * (3 * n + 1) * u
        for a, b in zip(got, ref):
            assert err(a, b) <= 2 * (5 * n + 5) * u
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, (h, *got)))
        first = (h, *got)


@pytest.mark.parametrize("learns", ["down.factors.0", "down.factors.1", "down.bias", "gate_up.bias", "norm.weight"])
def test_a_block_with_one_learning_parameter(learns):
    """The gradient of a parameter is the same whether the others learn or not."""
    torch.manual_seed(4)
    ff = KSGatedFeedForward(torch.bfloat16, "cuda", requires_grad=True)
    x, a, seed = (torch.randn(2, 50, 768, device="cuda").bfloat16() for _ in range(3))
    p = dict(ff.named_parameters())[learns]
    (want,) = torch.autograd.grad(ff(x, a), [p], seed)
    for other in ff.parameters():
        other.requires_grad_(other is p)
    out = ff(x, a)
    assert out.requires_grad
    (got,) = torch.autograd.grad(out, [p], seed)
    # (other kernels may run: the bound of a block's gradients in test_gpu_gated_block.py)
    assert err(got, want.double()) <= 72 * unit(torch.bfloat16)


@pytest.mark.parametrize("out_last", [False, True])
@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("rows,train", [(45, False), (512, False), (2560, False), (2560, True), (2309, True)])
def test_silu_down_to_the_smallest_numbers(rows, train, bs_last, out_last):
    """silu(g) between -86 and 10, where a bf16 result is a normal number, element by element, with values of every size
    next to one another.  The gate is exact (one product by 1); g log2(e), below 125, is rounded to 2^-18, 2^-18.5 of
    the result; exponential, reciprocal and four products 2^-20; the result 2^-8."""
    layer, x = layer_and_input([(1, 256, 64, 1)], torch.bfloat16, bs_last, out_last, rows, "silu", train=train)
    with torch.no_grad():
        layer.factors[0].zero_()
        layer.factors[0][:64].copy_(torch.eye(64, device="cuda").repeat(1, 4))   # the gate: feature j takes input j mod 64
        layer.bias.zero_()
        layer.bias.view(-1)[256:] = 1                                            # the up projection: 1
        x.uniform_(-86, 10)
        x[torch.rand(x.shape, device="cuda") < 0.3] *= 0.02
    got = layer(x)
    assert got.requires_grad == train
    g = (x if bs_last else x.t()).double().repeat(4, 1)
    want = g / (1 + torch.exp(-g))
    got = (got if out_last else got.t()).double()
    assert ((got - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * want.abs()).all()


def compare(layer, x, act, out_last):
    """Forward pass without and with gradients, and every gradient, against the definition."""
    n, u = len(layer.patterns), unit(layer.dtype)
    batch = x.numel() // layer.in_size
    seed = torch.randn(*((layer.out_size, batch) if out_last else (batch, layer.out_size)), device="cuda").to(layer.dtype)
    want, ref = exact_gradients(layer, x, seed, act, out_last)
    with torch.no_grad():
        assert err(layer(x), want) <= 2 * (3 * n + 1) * u
    leaf = x.detach().clone().requires_grad_(True)
    h = layer(leaf)
    assert err(h, want) <= 2 * (3 * n + 1) * u
    for i, (a, b) in enumerate(zip(torch.autograd.grad(h, [leaf, *params_of(layer)], seed), ref)):
        assert err(a, b) <= 2 * (5 * n + 5) * u, i


def gates_away_from_zero(layer):
    """Gate biases of 6 and -6, ten deviations of the gates around them: no rounding turns a gate's sign."""
    with torch.no_grad():
        half = layer.bias.view(2, -1)[0]
        half.copy_(torch.where(torch.rand(half.shape, device="cuda") < 0.5, -6.0, 6.0))


RAGGED = {"b136": [(4, 96, 96, 1), (1, 136, 96, 4)], "b264": [(2, 64, 64, 1), (1, 264, 64, 2)], "b392": [(2, 392, 192, 1)]}


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("act", ["silu", "sigmoid", "relu", "gelu", None])
@pytest.mark.parametrize("patterns", list(RAGGED))
@pytest.mark.parametrize("batch", [2304, 2309])
def test_features_that_fill_no_tile(batch, patterns, act, bs_last, out_last):
    """Tiles of 128 features of which the last has 8."""
    layer, x = layer_and_input(RAGGED[patterns], torch.bfloat16, bs_last, out_last, batch, act, train=True)
    if act == "relu":
        gates_away_from_zero(layer)
    compare(layer, x, act, out_last)


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("act", ["silu", "sigmoid", "relu", "gelu", None])
@pytest.mark.parametrize("patterns,batch", [([(1, 512, 192, 4)], 12301), ([(1, 392, 160, 8)], 6200), ([(2, 200, 192, 4)], 12304),
                                            ([(4, 512, 192, 1)], 12304), ([(1, 512, 136, 8)], 6147)])
def test_two_ctas(patterns, batch, act, bs_last, out_last):
    """Two CTAs of a cluster share a tile of 256 features (many tiles, blocks of 129 to 192 inputs): the second one of a
    last pair with all, 72 or 8 of its features; rows that a tensor map addresses or not; a pass over k that ends
    inside a chunk; with one block per feature group also a batch-first input."""
    layer, x = layer_and_input(patterns, torch.bfloat16, bs_last, out_last, batch, act, train=True)
    if act == "relu":
        gates_away_from_zero(layer)
    compare(layer, x, act, out_last)


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch", [45, 264])
def test_gradient_of_relu(batch, dtype, bs_last, out_last):
    layer, x = layer_and_input([(6, 64, 64, 1), (1, 512, 192, 2)], dtype, bs_last, out_last, batch, "relu", train=True)
    gates_away_from_zero(layer)
    compare(layer, x, "relu", out_last)


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("factors", [4, 5, 8, 9, 16])
def test_long_chains(factors, dtype, bs_last, out_last):
    """(Weights of a factor are scaled to keep a vector's size.  Layouts are planned up to eight factors.)"""
    patterns = ([(1, 8, 8, 8), (8, 8, 8, 1)] * 8)[:factors - 1] + [(1, 96, 64, 1)]
    layer, x = layer_and_input(patterns, dtype, bs_last, out_last, 77, "silu", train=True)
    with torch.no_grad():
        for f in layer.factors:
            f.mul_(3 ** 0.5)
    compare(layer, x, "silu", out_last)


def test_gradients_along_themselves():
    """fp32, by central differences in the direction of each gradient, where the slope is the gradient's norm.  With a
    unit direction and a step of 2^-4 an element moves by at most 0.01 or so: the truncation, step^2 / 6 of the third
    derivative, is 2e-5 times the ratio of third to first derivative (some tens for cubes and products of values near
    1).  The results' rounding, 1e-6 of 3e5 terms below 1 with random signs, is 1e-3 over twice the step, 1e-2; the
    gradients' norms are above 30.  Together below 1e-3 of the norm."""
    torch.manual_seed(3)
    layer = kb.KSGatedLinear([(6, 64, 64, 1), (1, 512, 192, 2)], dtype=torch.float32, requires_grad=True)
    rows = lambda *s: torch.randn(*s, device="cuda", requires_grad=True)
    args = (rows(300, 384), rows(300, 384), rows(384), rows(3, 384), *layer.parameters())

    def f(x, y, w, sc, *params):
        with torch.no_grad():
            for p, v in zip(layer.parameters(), params):
                p.copy_(v)
        z, n = kb.residual_norm(x, y, norm="rms", post_norm="layer", weight=w, scale=sc, gate=w, alpha=0.75)
        return layer(n).double().pow(2).sum() + z.double().pow(3).sum() * 0.1

    start = [a.detach().clone() for a in args]
    grads = torch.autograd.grad(f(*args[:4], *start[4:]), args)
    step = 2.0 ** -4
    for i, g in enumerate(grads):
        size = g.double().norm().item()
        assert size > 30
        v = g / size
        with torch.no_grad():
            plus = f(*[t + step * v if j == i else t for j, t in enumerate(start)])
            minus = f(*[t - step * v if j == i else t for j, t in enumerate(start)])
        slope = ((plus - minus) / (2 * step)).item()
        assert abs(slope - size) <= 1e-3 * size, (i, slope, size)


def test_gradients_through_a_network():
    """Every learning parameter of a network of gated blocks gets a finite gradient that is not 0."""
    torch.manual_seed(5)
    net = KSViTB(dtype=torch.bfloat16, depth=2, gated_mlp=True)
    for p in net.parameters():
        p.requires_grad_(True)
    net(torch.randn(2, 3, 224, 224, device="cuda").bfloat16()).float().pow(2).mean().backward()
    for name, p in net.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad.float()).all() and p.grad.float().norm() > 0, name


class Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


@pytest.mark.parametrize("how", ["pruned", "parametrised", "replaced"])
def test_factors_that_are_not_plain_parameters(how):
    """The layer computes with what its ParameterList gives, factor by factor (all of one shape here)."""
    torch.manual_seed(6)
    layer = kb.KSGatedLinear([(1, 64, 64, 1)] * 3, dtype=torch.float32, requires_grad=True)
    x = torch.randn(33, 64, device="cuda")
    before = layer(x).detach()
    if how == "pruned":
        torch.nn.utils.prune.random_unstructured(layer.factors, "0", 0.5)
    elif how == "parametrised":
        torch.nn.utils.parametrize.register_parametrization(layer.factors, "1", Doubled())
    else:
        layer.factors[0] = torch.nn.Parameter(3 * layer.factors[0].detach())
    factors = [f.detach() for f in layer.factors]
    got = layer(x)
    assert torch.equal(got, kb.kernel.gated_layer(x, [f.requires_grad_(True) for f in factors], layer.patterns, False, layer.bias))
    assert not torch.allclose(got, before, rtol=1e-3, atol=1e-3)
    assert all(p.grad is None for p in layer.parameters())
    got.sum().backward()
    assert all(p.grad is not None for p in layer.parameters())
