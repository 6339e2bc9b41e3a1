"""Prompts of several tokens over 8-bit caches against the formula in 64 bits; tolerances as in test_gpu_cache.check: the codes enter
the products exactly, scales act in fp32, weights are rounded once (fp16: after the part of the scale that they carry)."""

import pytest
import torch

import ksmm_b200 as kb
from test_gpu_cache import DEV, attended, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (8, 2, 128), (4, 1, 256), (4, 2, 80), (40, 1, 64), (3, 3, 16), (96, 1, 96), (2, 1, 240)])
def test_prompts(heads, kv, dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    for page, window in ((16, None), (48, 37), (64, 300)):
        lengths, new = [1, 300, 130, 257, 0, 64, 500, 40, 700], [1, 300, 1, 128, 0, 63, 129, 2, 65]
        cache, table, L, starts, q, _, _ = make(gen, lengths, new, heads, kv, dim, page, dtype, eight=True, tail=3)
        out = kb.cache_attention(q, cache, table, L, starts=starts, window=window)
        check(out[:-3], attended(q[:-3], cache, table, lengths, new, window=window), cache)
        assert (out[-3:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scales_of_any_size(dtype):
    """A sequence's scales over many powers of two, some negative or zero: values are bounded by the largest, which the error is taken of."""
    gen = torch.Generator().manual_seed(3)
    n, heads, kv, dim = 333, 8, 2, 64
    cache, table, L, _, q, _, _ = make(gen, [n], [n], heads, kv, dim, 16, dtype, eight=True)
    size = torch.exp2(torch.randint(-40, 1, cache.value_scales.shape, generator=gen).float()).to(DEV)
    sign = (torch.randint(0, 3, cache.value_scales.shape, generator=gen) - 1).float().to(DEV)
    cache.value_scales.mul_(size * sign)
    cache.key_scales.mul_(sign)
    ref = attended(q, cache, table, [n], [n])
    check(kb.cache_attention(q, cache, table, L), ref, cache)
    # as small as fp16 holds, and as large
    for by in (2.0 ** -12, 2.0 ** 12):
        cache.value_scales.mul_(by)
        out = kb.cache_attention(q, cache, table, L)
        unit = torch.finfo(dtype).eps / 2
        most = unit * ref.abs() * by + (2e-5 + unit) * 8 * by + (2.0 ** -25 * 2 if dtype == torch.float16 else 0)
        assert ((out.double() - ref * by).abs() <= most).all()
        cache.value_scales.div_(by)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_that_are_not_there_and_what_lies_behind(dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    lengths = [300, 300, 300]
    cache, table, L, starts, q, _, _ = make(gen, lengths, lengths, 4, 2, dim, 16, dtype, eight=True, width=40)
    ref = attended(q, cache, table, lengths, lengths)
    used = set(table[:, :19].flatten().tolist())
    for page in range(cache.pages):
        slots = slice(None) if page not in used else slice(300 % 16, None) if page in table[:, 18].tolist() else None
        if slots is not None:
            cache.keys.view(torch.uint8)[page, :, slots] = 127  # NaN
            cache.values.view(torch.uint8)[page, :, slots] = 127
            cache.key_scales[page, :, slots] = float("nan")
            cache.value_scales[page, :, slots] = float("inf")
    check(kb.cache_attention(q, cache, table, L), ref, cache)
    table[1, 10] = cache.pages  # not there: tokens 160 to 175
    table[2, 0] = -1
    out = kb.cache_attention(q, cache, table, L)
    check(out[:460], ref[:460], cache)
    assert torch.isnan(out[460:]).all()
    # a window that has left the page behind
    out = kb.cache_attention(q, cache, table, L, window=20)
    seen = attended(q, cache, table.clamp(0, cache.pages - 1), lengths, lengths, window=20)
    check(out[:460], seen[:460], cache)
    assert torch.isnan(out[460:460 + 20 + 15]).all() and torch.isnan(out[600:620]).all()
    check(out[460 + 35:600], seen[460 + 35:600], cache)
    check(out[600 + 35:], seen[600 + 35:], cache)
    assert torch.equal(out[:460], kb.cache_attention(q, cache, table, L, window=20)[:460])
