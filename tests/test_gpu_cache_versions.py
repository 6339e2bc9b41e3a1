"""Tensors that the cache calls write count as changed in place, through the extension module and without it."""

import pytest
import torch

import ksmm_b200 as kb
from ksmm_b200 import attention
from test_gpu_cache import DEV, make

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["native", "python"])
def native(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(attention, "_native", None)
    return request.param


@pytest.mark.parametrize("eight", [False, True])
def test_versions(eight, native):
    gen = torch.Generator().manual_seed(0)
    cache, table, L, _, q, k, v = make(gen, [20, 33], [4, 4], 4, 2, 64, 16, torch.float16, eight=eight)
    written = [cache.keys, cache.values] + ([cache.key_scales, cache.value_scales] if eight else [])
    read = [table, L, q, k, v]

    def versions(ts):
        return [t._version for t in ts]

    before, others = versions(written), versions(read)
    there = torch.empty_like(q)
    kb.cache_append(cache, table, L, k, v, q=q, q_out=there)
    assert versions(written) == [n + 1 for n in before] and there._version == 1
    kb.cache_append(cache, table, L, k, v)
    out = kb.cache_attention(q, cache, table, L)
    assert versions(written) == [n + 2 for n in before] and out._version == 0
    kb.cache_attention(q, cache, table, L, out=there)
    assert there._version == 2 and versions(read) == others
    kb.cache_attention(there, cache, table, L, out=there)
    assert there._version == 3
    with pytest.raises(ValueError):
        kb.cache_attention(q, cache, table, L, out=there[:, :2])
    assert there._version == 3


def test_a_graph_that_kept_the_output(native):
    """A norm keeps its input for the backward pass; attention that writes over it makes that raise instead of changing gradients."""
    gen = torch.Generator().manual_seed(0)
    cache, table, L, _, q, _, _ = make(gen, [20, 33], [4, 4], 4, 2, 64, 16, torch.float32)
    x = torch.randn(8, 256, device=DEV)
    weight = torch.ones(256, device=DEV, requires_grad=True)
    kb.residual_norm(x, weight=weight).sum().backward()
    h = kb.residual_norm(x, weight=weight)
    kb.cache_attention(q, cache, table, L, out=x.view(8, 4, 64))
    with pytest.raises(RuntimeError, match="inplace operation"):
        h.sum().backward()


def test_inference_tensors(native):
    gen = torch.Generator().manual_seed(0)
    with torch.inference_mode():
        cache, table, L, _, q, k, v = make(gen, [20, 33], [4, 4], 4, 2, 64, 16, torch.float16)
        there = torch.empty_like(q)
        kb.cache_append(cache, table, L, k, v, q=q, q_out=there)
        ref = kb.cache_attention(there, cache, table, L, out=torch.empty_like(q))
    # (and outside)
    kb.cache_append(cache, table, L, k, v, q=q, q_out=there)
    assert torch.equal(kb.cache_attention(there, cache, table, L, out=torch.empty_like(q)), ref)
