"""Paths of residual_norm's kernels that test_gpu_norm.py does not single out."""
import os
import subprocess
import sys

import pytest
import torch

import ksmm_b200 as kb
from test_gpu_norm import EVERY, PARAMS, check, definition, make, unit

pytestmark = pytest.mark.gpu

THREADS = """
import threading, torch
import ksmm_b200 as kb
torch.zeros(1, device="cuda")
# shared memory of these calls: 55 to 221 KB (batch-last), 28 to 192 KB (batch-first rings)
calls = [(c, 40, True) for c in (384, 1536, 500, 1001, 768, 1200)] + [(c, 1300, False) for c in (8192, 1152, 4096, 2048, 7000, 3000)]
xs = [torch.randn(*((c, n) if last else (n, c)), device="cuda", dtype=torch.bfloat16) for c, n, last in calls]
torch.cuda.synchronize()
start, failed, got = threading.Barrier(len(calls)), [], {}
def work(i):
    try:
        start.wait()
        for _ in range(20):
            got[i] = kb.residual_norm(xs[i], xs[i], bs_last=calls[i][2])
    except Exception as e:
        failed.append((calls[i], repr(e)))
threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
[t.start() for t in threads]; [t.join() for t in threads]
torch.cuda.synchronize()
assert not failed, failed
for i, x in enumerate(xs):
    for a, b in zip(got[i], kb.residual_norm(x, x, bs_last=calls[i][2])):
        assert torch.equal(a, b)
print("ok")
"""


def test_first_calls_of_many_widths_from_many_threads():
    """The shared memory that a kernel may ask for is settled by its first call, whichever width and thread that has."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for _ in range(3):
        res = subprocess.run([sys.executable, "-c", THREADS], cwd=root, capture_output=True, text=True, timeout=300)
        assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stderr[-3000:]


@pytest.mark.parametrize("bs_last", [False, True])
@pytest.mark.parametrize("channels,rows", [(64, 300), (256, 300), (1024, 90), (2048, 24), (256, 3000)])
@pytest.mark.parametrize("where", ["pre", "post"])
def test_gradients_far_from_zero(where, channels, rows, bs_last):
    """fp32 rows whose mean is some 3000 deviations.  Values are whole numbers near 2^14 and the sum of every 64 channels is a
    multiple of 64, so that partial sums (integers up to 2^24, multiples of 64 beyond), the mean (the channels
    are a power of two) and the differences from it are exact in fp32.  What is left are the deviation's rounding and the
    chains that test_gpu_norm.py counts, 128 u32; doubled, because the seeds have a mean that the gradient takes off."""
    g = torch.Generator(device="cuda").manual_seed(11)
    x = 16384 + (2 * torch.randn(rows, channels, device="cuda", generator=g)).round()
    groups = x.view(rows, -1, 64)
    groups[..., -1] -= groups.sum(-1) % 64
    w = torch.randn(channels, device="cuda", generator=g) + 1
    seed = torch.randn(rows, channels, device="cuda", generator=g) + 1
    lay = (lambda t: t.t().contiguous()) if bs_last else (lambda t: t)
    base = torch.zeros_like(x)

    def grads(v, weight, run):
        v, weight = (t.clone().requires_grad_(True) for t in (v, weight))
        return torch.autograd.grad(run(v, weight), [v, weight], lay(seed).to(v.dtype))

    def ours(v, weight):
        if where == "pre":
            return kb.residual_norm(v, weight=weight, bs_last=bs_last)
        return kb.residual_norm(lay(base), v, norm=None, post_norm="layer", post_weight=weight, bs_last=bs_last)

    def exact(v, weight):
        v = lay(v)
        d = v - v.mean(-1, keepdim=True)
        return lay(d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * weight)

    for a, b in zip(grads(lay(x), w, ours), grads(lay(x.double()), w.double(), exact)):
        assert ((a.double() - b).norm() / b.norm()).item() <= 256 * 2.0 ** -24


@pytest.mark.parametrize("channels", [8193, 2 ** 31, 2 ** 32 + 768])
def test_more_channels_than_the_library_takes(channels):
    """(The last one would reach the library as 768 channels.)"""
    for x, last in ((torch.zeros(1, 1, device="cuda", dtype=torch.float16).expand(1, channels), False),
                    (torch.zeros(1, 1, device="cuda", dtype=torch.float16).expand(channels, 1), True)):
        with pytest.raises((ValueError, kb.KsmmError), match="channels"):
            kb.residual_norm(x, bs_last=last)


@pytest.mark.parametrize("alpha", [-1.25, 0.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,bs_last", [((45, 96), False), ((45, 1303), False), ((2400, 768), False), ((601, 2304), False),
                                           ((9, 8192), False), ((384, 70), True), ((1000, 33), True), ((2304, 66), True)])
def test_scaled_streams(shape, bs_last, dtype, alpha):
    """alpha in every kernel: rows by groups, single elements, resident blocks, wide rows, columns, turned columns."""
    check(dtype, shape, norm="layer", post_norm="rms", bs_last=bs_last, samples=1, keys=EVERY, alpha=alpha)
    check(dtype, shape, norm="rms", bs_last=bs_last, keys=("weight", "shift"), alpha=alpha)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm,post_norm", [("layer", None), ("layer", "layer"), ("rms", "rms")])
@pytest.mark.parametrize("shape,bs_last,samples", [((300, 768), False, 3), ((301, 720), False, 1), ((40, 1480), False, 2),
                                                   ((45, 333), False, 1), ((66, 4096), False, 2), ((8, 8192), False, 1),
                                                   ((30, 5003), False, 1), ((768, 300), True, 3), ((2304, 66), True, 2)])
def test_gradients_know_the_unrounded_stream(shape, bs_last, samples, norm, post_norm, dtype):
    """z is 20 deviations from 0 (layer norms), where its rounding is off by 20 u of a deviation.  The statistics and the h of
    the forward pass are those of the unrounded z, so are the gradients: every result is rounded once, u; before that
    64 u32 for a chain, times 20 for the differences from the mean, times 4 for the gradient's own (its seeds have
    a mean of one deviation, and the sums over tokens add up such terms)."""
    x, y, p = make(dtype, shape, bs_last, samples, EVERY if post_norm else ("weight", "bias", "scale", "shift", "gate"), True, seed=2)
    if norm == "layer":
        x = x + 20
        if post_norm is None:
            y, p["gate"] = y + 4, 1 + p["gate"] / 4
    t = {k: v for k, v in {"x": x, "y": y, **p}.items() if v is not None}
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    exact = {k: v.double().requires_grad_(True) for k, v in t.items()}
    _, h = kb.residual_norm(leaves["x"], leaves["y"], norm=norm, post_norm=post_norm, alpha=0.75, bs_last=bs_last,
                            **{k: v for k, v in leaves.items() if k not in "xy"})
    _, want = definition(exact["x"], exact["y"], {k: exact.get(k) for k in PARAMS}, norm, post_norm, 0.75, 1e-5, bs_last)
    seed = (torch.randn(shape, device="cuda") + 1).to(dtype)
    got = torch.autograd.grad(h, list(leaves.values()), seed)
    ref = torch.autograd.grad(want, list(exact.values()), seed.double())
    for k, a, b in zip(leaves, got, ref):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= unit(dtype) + 64 * 20 * 4 * 2.0 ** -24, (k, off)


NARROW = """
import torch
import ksmm_b200 as kb
for dtype in (torch.float32, torch.float16, torch.bfloat16):
    for c in (300, 312, 327, 328, 336, 341, 342, 350):
        x = torch.randn(c, 40, device="cuda").to(dtype).requires_grad_(True)
        _, h = kb.residual_norm(x, x, bs_last=True)
        h.sum().backward()
torch.cuda.synchronize()
kb.check_device()
print("ok")
"""


def test_first_calls_at_the_limit_of_undeclared_shared_memory():
    """Batch-last calls of 328 to 341 channels take 46 to 48 KB beside the kernel's own 2: the first ones of a process."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", NARROW], cwd=root, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stderr[-3000:]
