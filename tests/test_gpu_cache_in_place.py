"""Results over their inputs: ``q_out`` and ``out`` may be q itself."""

import pytest
import torch

import ksmm_b200 as kb
from test_gpu_cache import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page", [(6, 6, 64, 16), (8, 2, 128, 64), (4, 1, 256, 16), (4, 4, 33, 5), (40, 1, 80, 16)])
def test_in_place(heads, kv, dim, page, dtype, eight):
    gen = torch.Generator().manual_seed(dim)
    for new in ([1] * 5, [1, 7, 300, 0, 64]):
        lengths = [1, 9, 300, 20, 2000]
        cache, table, L, starts, q, k, v = make(gen, lengths, new, heads, kv, dim, page, dtype, eight=eight)
        frequencies = kb.rotary_frequencies(dim // 2)
        for interleaved in (False, True):
            ref = kb.cache_append(cache, table, L, k, v, q=q, starts=starts, frequencies=frequencies, interleaved=interleaved)
            there = q.clone()
            assert kb.cache_append(cache, table, L, k, v, q=there, starts=starts, frequencies=frequencies, interleaved=interleaved,
                                   q_out=there) is there
            assert torch.equal(there, ref)
        ref = kb.cache_attention(q, cache, table, L, starts=starts)
        there = q.clone()
        assert kb.cache_attention(there, cache, table, L, starts=starts, out=there) is there
        assert torch.equal(there, ref)
