"""Table entries outside the pool, whatever their value: rows that need such a page are NaN, all others are as without it.

Tolerances as in test_gpu_cache.check."""

import pytest
import torch

import ksmm_b200 as kb
from test_gpu_cache import TYPES, attended, check, make

pytestmark = pytest.mark.gpu
ENTRIES = [-1, -2, -3, -2 ** 31, "pages", 2 ** 31 - 1]


@pytest.mark.parametrize("dtype,eight", [(t, e) for t in TYPES for e in (False, True)])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (6, 6, 64, 64), (4, 1, 256, 16), (4, 2, 96, 32), (4, 4, 33, 5)])
@pytest.mark.parametrize("lengths,new", [([300] * 3, [1] * 3), ([2900, 300, 3000], [1, 2, 1]), ([300] * 3, [70] * 3)])
def test_entries_outside_the_pool(lengths, new, heads, kv, dim, page, dtype, eight):
    gen = torch.Generator().manual_seed(dim + page)
    cache, table, L, starts, q, _, _ = make(gen, lengths, new, heads, kv, dim, page, dtype, eight=eight)
    ref = attended(q, cache, table, lengths, new)
    nth = 150 // page
    there = table[1, nth].clone()
    rows = slice(new[0], new[0] + new[1])
    others = [slice(0, new[0]), slice(new[0] + new[1], None)]
    # a window that has left the page behind, and one that still reaches it
    past = 300 - new[1] - (nth + 1) * page + 1
    seen = attended(q, cache, table, lengths, new, window=past)
    for entry in ENTRIES:
        table[1, nth] = cache.pages if entry == "pages" else entry
        out = kb.cache_attention(q, cache, table, L, starts=starts)
        assert torch.isnan(out[rows]).all(), entry
        for other in others:
            check(out[other], ref[other], cache)
        check(kb.cache_attention(q, cache, table, L, starts=starts, window=past), seen, cache)
        out = kb.cache_attention(q, cache, table, L, starts=starts, window=past + 1)
        assert torch.isnan(out[rows][0]).all()
        if new[1] > 1:
            check(out[rows][1:], attended(q, cache, table.index_put((torch.tensor(1), torch.tensor(nth)), there), lengths, new,
                                          window=past + 1)[rows][1:], cache)
    kb.check_device()


@pytest.mark.parametrize("dtype,eight", [(t, e) for t in TYPES for e in (False, True)])
def test_nothing_is_stored(dtype, eight):
    gen = torch.Generator().manual_seed(1)
    cache, table, L, starts, _, k, v = make(gen, [40, 40], [40, 8], 4, 2, 64, 16, dtype, eight=eight)
    names = ["keys", "values"] + (["key_scales", "value_scales"] if eight else [])
    before = {n: getattr(cache, n).clone() for n in names}
    for entry in ENTRIES:
        bad = torch.full_like(table, cache.pages if entry == "pages" else entry)
        kb.cache_append(cache, bad, L, k, v, starts=starts)
    for n in names:
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (before[n], getattr(cache, n)))
        assert torch.equal(a, b)
    kb.check_device()
