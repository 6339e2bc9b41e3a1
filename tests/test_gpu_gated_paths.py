"""Paths of the gated layer's kernels against the definition in 64 bits.

Tolerances are those of test_gpu_gated.py (n factors, u = eps / 2 of the type, relative 2-norms): 2 (3 n + 1) u forward,
2 (5 n + 5) u backward.
"""
import pytest
import torch

from ksmm_b200.ksvit import KSGatedFeedForward
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
@pytest.mark.parametrize("patterns", [[(1, 512, 64, 8)], [(2, 96, 64, 16)]], ids=["pairs", "one_tile"])
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
