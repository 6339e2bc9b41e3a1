"""Paths of residual_norm's kernels that test_gpu_norm.py does not single out."""
import os
import subprocess
import sys

import pytest
import torch

import ksmm_b200 as kb

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
