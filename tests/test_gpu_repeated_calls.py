"""The same call gives the same bits, however busy an SM's memory pipes are.

Shapes whose results are stored element by element keep the pipes full, so that loads from a staging buffer may wait
there for longer than the copy that refills it takes: every kernel that hands such a buffer back waits for its loads.
(Without that wait about one call in a hundred of the first shape had a warp's results off.)
"""
import pytest
import torch

import ksmm_b200 as kb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pattern,batch,bs_last,dtype", [
    ((1, 88, 126, 24), 13509, True, torch.float32), ((4, 60, 64, 8), 9001, True, torch.float32),
    ((2, 52, 96, 2), 20001, False, torch.float32), ((1, 132, 80, 4), 9999, False, torch.float32),
    ((1, 192, 192, 2), 12545, False, torch.float16), ((1, 192, 96, 4), 12545, False, torch.bfloat16)])
def test_one_factor(pattern, batch, bs_last, dtype):
    torch.manual_seed(0)
    a, b, c, d = pattern
    w = torch.randn(a * d * c, b, device="cuda").to(dtype)
    x = torch.randn(*((a * c * d, batch) if bs_last else (batch, a * c * d)), device="cuda").to(dtype)
    first = kb.forward_ex(x, w, bs_last, *pattern)
    other = torch.zeros(1, dtype=torch.long, device="cuda")
    for _ in range(600):
        other += (kb.forward_ex(x, w, bs_last, *pattern) != first).any()
    assert other.item() == 0
    kb.check_device()


@pytest.mark.parametrize("kind", ["gated", "layer"])
def test_gradients(kind):
    torch.manual_seed(1)
    patterns = [(6, 8, 16, 3), (4, 88, 6, 6), (1, 126, 88, 24)]
    make = kb.KSGatedLinear if kind == "gated" else kb.KSLinear
    layer = make(patterns, bias=False, dtype=torch.float32, bs_last=True, requires_grad=True)
    x = torch.randn(288, 13509, device="cuda", requires_grad=True)
    h = layer(x)
    seed = torch.randn_like(h)
    step = lambda: torch.autograd.grad(h, [x, *layer.factors], seed, retain_graph=True)
    first = step()
    other = torch.zeros(1, dtype=torch.long, device="cuda")
    for _ in range(200):
        for p, q in zip(step(), first):
            other += (p != q).any()
    assert other.item() == 0


@pytest.mark.parametrize("rows,channels", [(12545, 768), (4001, 4096), (3001, 2048)])
def test_norms(rows, channels):
    torch.manual_seed(2)
    x, y = (torch.randn(rows, channels, device="cuda").bfloat16() for _ in range(2))
    first = kb.residual_norm(x, y, post_norm="rms")
    other = torch.zeros(1, dtype=torch.long, device="cuda")
    for _ in range(300):
        for p, q in zip(kb.residual_norm(x, y, post_norm="rms"), first):
            other += (p != q).any()
    assert other.item() == 0
