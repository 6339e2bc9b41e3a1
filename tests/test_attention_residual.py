"""KSAttention refuses a residual that requires a gradient, as it refuses such an input: the sum would lose it.  No GPU."""
import pytest
import torch

import ksmm_b200 as kb

Q = [(6, 64, 64, 1), (1, 192, 192, 2)]


def test_a_residual_that_requires_a_gradient():
    attn = kb.KSAttention(Q, Q, 6, device="meta")
    x = torch.zeros(2, 1, 384, dtype=torch.float16)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="residual requires a gradient"):
        attn(x, None, n[:, None], n, residual=x.clone().requires_grad_())
    with pytest.raises(ValueError, match="x requires a gradient"):
        attn(x.clone().requires_grad_(), None, n[:, None], n)
