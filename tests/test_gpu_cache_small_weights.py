"""Rows whose weight lies on one key with a value of 0, while thousands of others, 17 nats below it, make the result: none of
them may vanish in the 16 bits that the products take.

Tolerance, relative to the sum of |weight * value| (all values but the first are positive: the result itself): the scores
reach 24.5 in log2 units, whose rounding (a product, a scale, a difference) is 4 * 24.5 * 2^-24 < 6e-6 of a weight, and those of the
others' own sums of dim products below (dim + 8) 2^-24 * |q| |k| * scale < 3e-5: 4e-5 with ex2's 2^-22.  Weights are rounded once
where prompts or a bf16 model on an 8-bit cache take them as one 16-bit number: u16 of each.  fp16 numbers are subnormal
below 2^-14: the weights are held such that the row's largest is 2^10 at least, so that they are off by at most 2^-35 of it,
`length` of them times values of up to 320.  Then the result's own rounding, half a step of 2^-24 in fp16 at least.
"""
import pytest
import torch

import ksmm_b200 as kb
from test_gpu_cache import DEV, TYPES, attended, make, unit

pytestmark = pytest.mark.gpu


def dominated(gen, length, new, heads, kv, dim, dtype, eight):
    """A sequence whose first key scores 17 (after the scale) with every new token, and has values of 0."""
    cache, table, L, _, q, _, _ = make(gen, [length], [new], heads, kv, dim, 64, dtype, eight=eight)
    q.mul_(0.5)
    q[..., 0] = 8.0
    shape = (cache.pages, kv, 64, dim)
    keys, values = 0.5 * torch.randn(shape, generator=gen), 256 * (1 + 0.25 * torch.rand(shape, generator=gen))
    keys[..., 0] *= 0.5
    first = table[0, 0].item()
    keys[first, :, 0] = 0
    keys[first, :, 0, 0] = 17.0 * dim ** 0.5 / 8
    values[first, :, 0] = 0
    for t, to, scales in ((keys, cache.keys, cache.key_scales), (values, cache.values, cache.value_scales)):
        if eight:
            s = (t.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
            scales.copy_(s)
            to.view(torch.uint8).copy_((t / s[..., None]).to(torch.float8_e4m3fn).view(torch.uint8))
        else:
            to.copy_(t)
    return cache, table, L, q


# (prompts over 131072 tokens with 64 columns: the others take the same path as over 8192)
CALLS = [(length, new, *heads) for length, new in ((500, 1), (1000, 2), (8192, 1), (8192, 3), (131072, 1), (700, 200), (8192, 150))
         for heads in ((2, 2, 64), (8, 2, 128), (4, 1, 256))] + [(131072, 130, 2, 2, 64)]


@pytest.mark.parametrize("dtype,eight", [(t, e) for t in TYPES for e in (False, True) if not (e and t == torch.float32)])
@pytest.mark.parametrize("length,new,heads,kv,dim", CALLS)
def test_a_key_that_takes_the_weight(length, new, heads, kv, dim, dtype, eight):
    gen = torch.Generator().manual_seed(length + new + dim)
    cache, table, L, q = dominated(gen, length, new, heads, kv, dim, dtype, eight)
    ref = attended(q, cache, table, [length], [new])
    out = kb.cache_attention(q, cache, table, L)
    once = dtype != torch.float32 and (new > 100 or (eight and dtype == torch.bfloat16))
    most = (unit(dtype) + 4e-5 + (unit(torch.float16 if eight and new <= 3 else dtype) if once else 0)) * ref.abs()
    if dtype == torch.float16 or eight:
        most = most + length * 2.0 ** -35 * 320
    if dtype == torch.float16:
        most = most + 2.0 ** -25
    off = (out.double() - ref).abs()
    assert (off <= most).all(), (off / most).max().item()
    kb.check_device()
