"""KSAttention and a block around it, as a generating model uses them: prompts, then token by token.

Tolerances: projections, attention and output layer each round to the layer's type once (u = eps / 2 of the value) from sums in
32 bits; the 8-bit cache adds half a step of e4m3, 2^-4, to each key and value.  In the relative 2-norm: q, k and v carry u each,
which shifts a score by 2 u |q| |k| * scale (below 8 u here) and a value by u; the output layer's input carries u again and its
result: 16 u bounds their sum, 2^-4 * 16 the 8-bit case.
"""
import pytest
import torch

import ksmm_b200 as kb
from ksmm_b200.ksvit import KSGatedFeedForward

pytestmark = pytest.mark.gpu
DEV = "cuda"
Q = [(6, 64, 64, 1), (1, 192, 192, 2)]    # 384 -> 384
KV = [(6, 64, 64, 1), (1, 64, 192, 2)]    # 384 -> 128


def unit(t):
    return torch.finfo(t).eps / 2


def dense(layer):
    w = layer.get_dense_product().double()
    return w, 0 if layer.bias is None else layer.bias.double().reshape(-1)


def rotated(t, position, frequencies):
    n = frequencies.shape[0]
    angle = position.double()[:, None, None] * frequencies
    x, y = t[..., :n], t[..., n:2 * n]
    return torch.cat([x * angle.cos() - y * angle.sin(), x * angle.sin() + y * angle.cos(), t[..., 2 * n:]], -1)


def plain(attn, x, window=None):
    """One sequence from its first token on, in 64 bits."""
    x = x.double()
    layers = list(attn.qkv.layers) if hasattr(attn, "qkv") else [attn.q, *attn.kv.layers]
    q, k, v = (x @ w.t() + b for w, b in map(dense, layers))
    n, d = x.shape[0], attn.head_dim
    q, k, v = (t.view(n, -1, d) for t in (q, k, v))
    at = torch.arange(n, device=x.device)
    if attn.frequencies is not None:
        q, k = rotated(q, at, attn.frequencies), rotated(k, at, attn.frequencies)
    k, v = (t.repeat_interleave(attn.heads // attn.kv_heads, 1) for t in (k, v))
    hidden = at[None] > at[:, None]
    if window:
        hidden = hidden | (at[None] <= at[:, None] - window)
    w = torch.softmax((torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5).masked_fill(hidden, -torch.inf), -1)
    a = torch.einsum("hqk,khd->qhd", w, v).reshape(n, -1)
    w, b = dense(attn.out)
    return a @ w.t() + b


def tables(lengths, page):
    """Pages in turn for sequences that may grow to `lengths`."""
    width = max(-(-n // page) for n in lengths)
    return torch.arange(len(lengths) * width, dtype=torch.int32, device=DEV).view(len(lengths), width), len(lengths) * width


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv,window,eight", [(None, None, False), (KV, None, False), (KV, 20, False), (KV, None, True)])
def test_prompts_and_tokens(kv, window, eight, dtype):
    if eight and dtype == torch.float32:
        pytest.skip("8 bits beside 16-bit models")
    torch.manual_seed(0)
    attn = kb.KSAttention(Q, Q, 6, kv_patterns=kv, dtype=dtype, device=DEV, window=window, rotary_dim=48)
    final = [70, 33, 129]
    prompts = [50, 1, 127]
    xs = [torch.randn(n, 384, device=DEV).to(dtype) for n in final]
    refs = [plain(attn, x, window) for x in xs]
    table, pages = tables(final, 16)
    cache = attn.new_cache(pages, 16, eight=eight)
    got = [[] for _ in final]
    # the prompts as one ragged batch, padded by four rows
    x = torch.cat([x[:n] for x, n in zip(xs, prompts)] + [torch.zeros(4, 384, device=DEV, dtype=dtype)])
    starts = torch.tensor([0, 50, 51, 178], dtype=torch.int32, device=DEV)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    y = attn(x, cache, table, lengths, starts=starts)
    for s in range(3):
        got[s].append(y[starts[s]:starts[s + 1]])
    # two tokens of each, then one by one until every sequence is done: padded batches, sequences that have ended wait
    now = list(prompts)
    while any(n < f for n, f in zip(now, final)):
        step = [min(2 if now == prompts else 1, f - n) for n, f in zip(now, final)]
        x = torch.cat([x[n:n + m] for x, n, m in zip(xs, now, step)])
        starts = torch.tensor([sum(step[:i]) for i in range(4)], dtype=torch.int32, device=DEV)
        now = [n + m for n, m in zip(now, step)]
        y = attn(x, cache, table, torch.tensor(now, dtype=torch.int32, device=DEV), starts=starts, max_new=2)
        for s in range(3):
            got[s].append(y[starts[s]:starts[s + 1]])
    most = 16 * (2.0 ** -4 if eight else unit(dtype) + 2.0 ** -22)
    for parts, ref in zip(got, refs):
        out = torch.cat(parts).double()
        assert out.shape == ref.shape and (out - ref).norm() / ref.norm() < most
    kb.check_device()


def test_residual_and_shapes():
    torch.manual_seed(1)
    attn = kb.KSAttention(Q, Q, 6, dtype=torch.bfloat16, device=DEV)
    x = torch.randn(2, 30, 384, device=DEV).bfloat16()
    table, pages = tables([30, 30], 64)
    cache = attn.new_cache(pages)
    lengths = torch.tensor([30, 30], dtype=torch.int32, device=DEV)
    y = attn(x, cache, table, lengths)
    z = attn(x, cache, table, lengths, residual=x)
    assert y.shape == z.shape == x.shape
    assert (z.double() - y.double() - x.double()).abs().max() <= 4 * unit(torch.bfloat16) * z.abs().max()
    with pytest.raises(ValueError, match="gradient"):
        attn(x.requires_grad_(), cache, table, lengths)
    assert attn(x.detach()[:, :0], cache, table, lengths * 0).shape == (2, 0, 384)
    attn.half()
    assert attn.frequencies.dtype == torch.float64


def test_blocks_in_a_graph():
    """Two blocks of attention and gated feed-forward; a captured step replayed as the sequences grow equals the prompt's rows."""
    torch.manual_seed(2)
    dtype, dim = torch.bfloat16, 768
    pats = [(4, 192, 192, 1), (1, 192, 192, 4)]
    blocks = [(kb.ResidualNorm(dim, norm="rms", dtype=dtype, device=DEV), kb.KSAttention(pats, pats, 12, dtype=dtype, device=DEV),
               KSGatedFeedForward(dtype, DEV, norm="rms")) for _ in range(2)]
    n = 24
    x = torch.randn(2, n, dim, device=DEV).to(dtype)
    table, pages = tables([n, n], 16)

    def run(x, caches, lengths):
        for (norm, attn, ff), cache in zip(blocks, caches):
            x = ff(x, attn(norm(x), cache, table, lengths))
        return x

    with torch.no_grad():
        full = run(x, [b[1].new_cache(pages, 16) for b in blocks], torch.tensor([n, n], dtype=torch.int32, device=DEV))
        caches = [b[1].new_cache(pages, 16) for b in blocks]
        token, lengths = torch.empty(2, 1, dim, device=DEV, dtype=dtype), torch.ones(2, dtype=torch.int32, device=DEV)
        token.copy_(x[:, :1])
        run(token, caches, lengths)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(token, caches, lengths)
        steps = []
        for t in range(n):
            token.copy_(x[:, t:t + 1])
            lengths.fill_(t + 1)
            graph.replay()
            steps.append(out.clone())
    steps = torch.cat(steps, 1)
    # the same sums in another order and through other kernels: eight roundings a block
    assert (steps.double() - full.double()).norm() / full.double().norm() < 16 * 2 * unit(dtype)
    kb.check_device()
