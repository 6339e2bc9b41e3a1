"""KSGatedLinear and gated_chain_forward against their definition in 64 bits, forward and backward.

Tolerances (relative 2-norm over a tensor).  One factor adds a relative error e: for 16-bit types the rounding of
its result, u = eps / 2 per element (sums are fp32), for fp32 at most 1e-6 (measured for the tensor-core kernel
up to c = 192: 5e-7 to 8e-7; FFMA kernels less).  A later factor with random weights passes a relative error on
without gain, on average over a vector; outputs of few elements may be twice off the average.  The gate's
function has a condition number |g act'(g) / act(g)| below 2 in the 2-norm for the gates here (normal, deviation
near 0.6).  So a half arrives with n e, the product with (2 + 1) n e, and rounding adds e:
forward (3 n + 1) e, doubled for short vectors.  Backward, dg = dh u act'(g) has the error of the kept halves
(rounded once more) through act' (condition below 2), (n + 1) e (1 + 2) + e, and passes n transposed factors, each
with an e for its result; weight gradients multiply that with intermediates of n e.  Together
(3 (n + 1) + 1 + n + n + 1) e = (5 n + 5) e, doubled for short vectors.
"""
import pytest
import torch

import ksmm_b200 as kb

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
BASE = [(4, 192, 192, 1), (1, 512, 192, 4)]
SMALL = [(6, 64, 64, 1), (1, 512, 192, 2)]
CHAIN3 = [(1, 64, 64, 16), (4, 64, 64, 4), (16, 176, 64, 1)]
ODD = [(2, 3, 5, 7), (1, 4, 6, 7)]
ONE = [(1, 96, 80, 3)]
WIDE_BLOCK = [(2, 136, 264, 1)]
LAYOUTS = [(False, False), (False, True), (True, True), (True, False)]


def unit(dtype):
    return 1e-6 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


ACT = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid,
       None: lambda t: t}


def definition(x, factors, bias, patterns, bs_last, out_last, act):
    n_out = patterns[-1][0] * patterns[-1][1] * patterns[-1][3]
    halves = []
    for q in range(2):
        y = x if bs_last else x.t()
        for (a, b, c, d), w in zip(patterns, factors):
            k = w.reshape(2, a, d, c, b)[q].permute(0, 3, 2, 1)
            y = torch.einsum("ijkl,ikln->ijln", k, y.reshape(a, c, d, -1)).reshape(a * b * d, -1)
        halves.append(y if bias is None else y + bias.reshape(2, n_out, 1)[q])
    h = ACT[act](halves[0]) * halves[1]
    return h if out_last else h.t()


def layer_and_input(patterns, dtype, bs_last, out_last, batch, act, bias=True, train=False, seed=0):
    torch.manual_seed(seed)
    layer = kb.KSGatedLinear(patterns, bias=bias, dtype=dtype, bs_last=bs_last, out_bs_last=out_last, activation=act,
                             requires_grad=train)
    x = torch.randn(*((layer.in_size, batch) if bs_last else (batch, layer.in_size)), device="cuda").to(dtype)
    return layer, x


def err(a, b):
    return ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()


def check(patterns, dtype, bs_last, out_last, batch, act="silu", bias=True, train=True):
    layer, x = layer_and_input(patterns, dtype, bs_last, out_last, batch, act, bias)
    params = list(layer.factors) + ([layer.bias] if bias else [])
    exact = [t.detach().double().requires_grad_(True) for t in (x, *params)]
    want = definition(exact[0], exact[1:1 + len(patterns)], exact[-1] if bias else None, patterns, bs_last, out_last, act)
    n = len(patterns)
    forward, backward = 2 * (3 * n + 1) * unit(dtype), 2 * (5 * n + 5) * unit(dtype)
    got = layer(x)
    assert tuple(got.shape) == tuple(want.shape) and got.dtype == dtype and got.is_contiguous()
    assert err(got, want) <= forward
    if not train:
        return
    for p in params:
        p.requires_grad_(True)
    leaf = x.clone().requires_grad_(True)
    h = layer(leaf)
    assert err(h, want) <= forward
    seed = torch.randn(want.shape, device="cuda", dtype=torch.float32).to(dtype)
    grads = torch.autograd.grad(h, [leaf, *params], seed)
    ref = torch.autograd.grad(want, exact, seed.double())
    for i, (a, b) in enumerate(zip(grads, ref)):
        assert a.shape == b.shape and a.dtype == dtype
        assert err(a, b) <= backward, (i, err(a, b), backward)
    kb.check_device()


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("patterns", [BASE, SMALL, CHAIN3, ODD, ONE, WIDE_BLOCK], ids=["base", "small", "chain3", "odd", "one", "wide"])
def test_patterns_types_layouts(patterns, dtype, bs_last, out_last):
    check(patterns, dtype, bs_last, out_last, 200)


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("batch", [1, 2, 7, 8, 16, 45, 127, 129, 197, 1003])
def test_batches(batch, bs_last, out_last):
    check(BASE, torch.bfloat16, bs_last, out_last, batch)


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("batch", [1, 7, 45, 197])
def test_batches_fp32(batch, bs_last, out_last):
    check(SMALL, torch.float32, bs_last, out_last, batch)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", None])
def test_activations(act, dtype):
    check(SMALL, dtype, False, True, 264, act=act)
    check(SMALL, dtype, True, True, 264, act=act, bias=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_relu(dtype):
    # (its gradient jumps at 0, where a rounded half may lie on the other side: the forward pass only)
    check(SMALL, dtype, False, False, 264, act="relu", train=False)


@pytest.mark.parametrize("batch", [3000, 6501])
def test_many_tiles(batch):
    for bs_last, out_last in LAYOUTS:
        check(SMALL, torch.float16, bs_last, out_last, batch, act="gelu")


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("batch", [33, 450, 1003])
def test_ragged_fp32_inference(batch, bs_last, out_last):
    """Padded intermediates go through the tensor-core kernel with their padding."""
    for patterns in (BASE, SMALL, CHAIN3):
        check(patterns, torch.float32, bs_last, out_last, batch, train=False)


@pytest.mark.parametrize("bs_last,out_last", LAYOUTS)
@pytest.mark.parametrize("patterns", [CHAIN3, [(2, 52, 64, 1)], [(2, 52, 64, 2)], [(3, 32, 52, 1), (1, 116, 96, 1)]],
                         ids=["chain3", "one", "interleaved", "second"])
@pytest.mark.parametrize("batch", [544, 1003])
def test_rows_of_weights_that_are_no_whole_pieces(batch, patterns, bs_last, out_last):
    """fp32 inference copies such weights for the tensor cores, what lies behind a row may be anything."""
    filler = torch.full((1 << 24,), float("nan"), device="cuda")
    del filler
    check(patterns, torch.float32, bs_last, out_last, batch, train=False)
