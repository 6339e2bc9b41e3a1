"""What the kernels for few rows keep beyond 16 bits, 8-bit caches with pages that are not there, and several tokens over long
sequences.

Tolerance of few rows: as in test_gpu_cache without the weights' own rounding, which enter the products in two parts: u of the
result and 2e-5 of the largest |v|.  A bf16 model on an 8-bit cache takes them as one fp16 number: 2^-11 of the largest |v| more.
"""
import pytest
import torch

import ksmm_b200 as kb
from test_gpu_cache import TYPES, attended, check, make, unit

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,eight", [(t, e) for t in TYPES for e in (False, True)])
@pytest.mark.parametrize("heads,kv,dim,page", [(6, 6, 64, 16), (8, 2, 128, 64), (4, 1, 256, 16), (16, 1, 128, 16), (4, 2, 80, 16), (2, 1, 33, 5)])
def test_weights_in_two_parts(heads, kv, dim, page, dtype, eight):
    gen = torch.Generator().manual_seed(heads + dim)
    # (few keys: their roundings do not average out)
    lengths, new = [2, 3, 5, 8, 30, 3000], [1, 2, 1, 2, 1, 1]
    cache, table, L, starts, q, _, _ = make(gen, lengths, new, heads, kv, dim, page, dtype, eight=eight)
    ref = attended(q, cache, table, lengths, new)
    out = kb.cache_attention(q, cache, table, L, starts=starts, max_new=2)
    if eight and dtype == torch.bfloat16:
        off = (out.double() - ref).abs()
        assert (off <= unit(dtype) * ref.abs() + (2e-5 + 2.0 ** -11) * 8.0).all()
    else:
        check(out, ref, cache, rounded_weights=False)


@pytest.mark.parametrize("dtype,eight", [(t, e) for t in TYPES for e in (False, True)])
@pytest.mark.parametrize("length,new", [(9000, 4), (20000, 16), (9000, 40), (20000, 100)])
def test_several_tokens_over_long_sequences(length, new, dtype, eight):
    gen = torch.Generator().manual_seed(length + new)
    for heads, kv, dim in ((8, 2, 128), (2, 2, 64), (2, 1, 256)):
        lengths, news = [length, 70, length // 3], [new, 1, new]
        cache, table, L, starts, q, _, _ = make(gen, lengths, news, heads, kv, dim, 64, dtype, eight=eight)
        for window in (None, 5000):
            out = kb.cache_attention(q, cache, table, L, starts=starts, window=window)
            check(out, attended(q, cache, table, lengths, news, window=window), cache)
