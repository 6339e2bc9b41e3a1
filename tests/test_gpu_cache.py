"""cache_append and cache_attention against their definitions in 64 bits.

Tolerances.  A result rounded once to type t is off by at most u = eps(t) / 2 of its own size.  Before that everything is fp32:
* append: one product pair and a sum on top of an angle that is exact to 2^-24: 4 u32 of the pair's norm, u32 = 2^-24;
  stored in 8 bits an element is off by half a step of e4m3 (2^-4 of its size, or 2^-10 of the scale below 2^-6), and where the
  quotient lies next to a border by as much on the other side: 2^-4 + 2 u32 bounds both;
* attention: a row is a mean of values with weights that sum to 1.  A score is off by (dim + 8) u32 |q| |k|, which the inputs
  keep below 64 in log2 units / 2^24 = 4e-6, so a weight by 8e-6 of itself (its score's error and the maximum's); sums over
  `length` keys in a tree of parts add (length / 32 + 64) u32; weights that enter a 16-bit product as two parts are off by
  u16^2.  Together below 2e-5 of max |v|, on top of the final rounding.  Where the weights are rounded once to the 16-bit type
  (prompts), each is off by u16 of itself: u16 of max |v| more.
"""
import math

import pytest
import torch

import ksmm_b200 as kb

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def unit(t):
    return torch.finfo(t).eps / 2


def make(gen, lengths, new, heads, kv, dim, page, dtype, eight=False, tail=0, spare=3, token_major=False, width=None):
    """A filled cache, its table (pages in no order, -1 behind the last) and the new tokens' q, k, v."""
    used = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(max(used), 1) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    shape = (pages, page, kv, dim) if token_major else (pages, kv, page, dim)
    keys, values = (torch.randn(shape, generator=gen) for _ in range(2))
    if token_major:
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    if eight:
        scales = [t.abs().amax(-1) / 448 for t in (keys, values)]
        keys, values = ((t / s[..., None]).to(F8).to(DEV) for t, s in zip((keys, values), scales))
        cache = kb.KVCache.of(keys, values, *(s.to(DEV) for s in scales))
    else:
        cache = kb.KVCache.of(keys.to(dtype).to(DEV), values.to(dtype).to(DEV))
    tokens = sum(new) + tail
    q, k, v = (torch.randn(tokens, h, dim, generator=gen).to(dtype).to(DEV) for h in (heads, kv, kv))
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    return cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), starts, q, k, v


def stored(cache, table, s, length):
    """The cache's keys and values of a sequence in 64 bits, (heads, length, dim)."""
    used = table[s, :-(-length // cache.page_size)].long()
    out = []
    for t, sc in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        t = (t.view(torch.uint8)[used].view(F8) if t.dtype == F8 else t[used]).double()
        if sc is not None:
            t = t * sc[used].double()[..., None]
        out.append(t.transpose(0, 1).flatten(1, 2)[:, :length])
    return out


def attended(q, cache, table, lengths, new, scale=None, window=None):
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group, at = q.shape[1] // cache.heads, 0
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for s, (length, n) in enumerate(zip(lengths, new)):
        if length > 0 and n > 0:
            k, v = stored(cache, table, s, length)
            k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
            q_at = torch.arange(length - n, length, device=q.device)[:, None]
            k_at = torch.arange(length, device=q.device)
            seen = k_at <= q_at
            if window:
                seen &= k_at > q_at - window
            x = (q[at:at + n].double().transpose(0, 1) @ k.transpose(1, 2)) * scale
            w = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
            out[at:at + n] = torch.where(seen.any(-1)[:, None, None], (w @ v).transpose(0, 1), 0.0)
        at += n
    return out


def check(out, ref, cache, rounded_weights=True):
    assert out.dtype in TYPES and not torch.isnan(out).any()
    top = 8.0  # (|v| of the inputs: randn)
    most = unit(out.dtype) * ref.abs() + 2e-5 * top + (unit(out.dtype) * top if rounded_weights and out.dtype != torch.float32 else 0)
    off = (out.double() - ref).abs()
    assert (off <= most).all(), (off / most).max().item()
    # most elements are far inside: the norm of the error shows a part that is missing
    if ref.norm() > 0:
        assert (out.double() - ref).norm() / ref.norm() < 4 * unit(out.dtype) + 2e-5


SHAPES = [  # heads, kv_heads, dim
    (6, 6, 64), (8, 2, 128), (8, 1, 256), (4, 4, 80), (6, 2, 96), (20, 1, 64), (3, 3, 24), (2, 1, 33), (48, 2, 128), (1, 1, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_one_token(heads, kv, dim, dtype):
    gen = torch.Generator().manual_seed(heads * dim)
    for page in (16, 64, 5):
        lengths = [1, 15, 16, 17, 0, 64, 65, 200, 3]
        new = [1] * len(lengths)
        cache, table, L, _, q, _, _ = make(gen, lengths, new, heads, kv, dim, page, dtype)
        out = kb.cache_attention(q, cache, table, L)
        check(out, attended(q, cache, table, lengths, new), cache)
        assert (out[4] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (8, 2, 128), (4, 1, 256), (4, 2, 80), (32, 2, 112), (4, 4, 20)])
def test_eight_bits(heads, kv, dim, dtype):
    gen = torch.Generator().manual_seed(heads + dim)
    for page in (16, 48):
        lengths = [1, 130, 77, 0, 1000]
        cache, table, L, _, q, _, _ = make(gen, lengths, [1] * 5, heads, kv, dim, page, dtype, eight=True)
        check(kb.cache_attention(q, cache, table, L), attended(q, cache, table, lengths, [1] * 5), cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [None, 1, 63, 64, 100, 5000])
def test_windows_and_long_sequences(window, dtype):
    gen = torch.Generator().manual_seed(5)
    lengths = [1, 64, 5000, 129, 1023]
    for new in ([1] * 5, [1, 2, 3, 4, 5]):
        cache, table, L, starts, q, _, _ = make(gen, lengths, new, 8, 2, 128, 32, dtype)
        out = kb.cache_attention(q, cache, table, L, starts=starts, window=window, max_new=max(new))
        check(out, attended(q, cache, table, lengths, new, window=window), cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (8, 2, 128), (4, 1, 256), (4, 2, 80), (40, 1, 64)])
def test_prompts(heads, kv, dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    for window in (None, 37):
        lengths, new = [1, 300, 130, 257, 0, 64, 500, 40], [1, 300, 1, 128, 0, 63, 129, 2]
        cache, table, L, starts, q, _, _ = make(gen, lengths, new, heads, kv, dim, 16, dtype, tail=3)
        out = kb.cache_attention(q, cache, table, L, starts=starts, window=window)
        check(out[:-3], attended(q[:-3], cache, table, lengths, new, window=window), cache)
        assert (out[-3:] == 0).all()
        there = torch.full_like(q, 7.0)
        assert kb.cache_attention(q, cache, table, L, starts=starts, window=window, out=there, max_new=2) is there
        check(there[:-3], attended(q[:-3], cache, table, lengths, new, window=window), cache)
        assert (there[-3:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_prompts_and_more_rows_than_tokens(dtype):
    gen = torch.Generator().manual_seed(11)
    cache, table, L, _, q, _, _ = make(gen, [200, 200, 200], [100] * 3, 4, 2, 64, 16, dtype)
    check(kb.cache_attention(q, cache, table, L), attended(q, cache, table, [200] * 3, [100] * 3), cache)
    # tokens before a sequence's first: no key to see
    short = torch.tensor([60, 100, 0], dtype=torch.int32, device=DEV)
    out = kb.cache_attention(q, cache, table, short, scale=0.25)
    check(out, attended(q, cache, table, [60, 100, 0], [100] * 3, scale=0.25), cache)
    assert (out[:40] == 0).all() and (out[200:] == 0).all()


def rotated(t, position, frequencies, interleaved):
    t = t.double()
    if frequencies is None:
        return t
    n = frequencies.shape[0]
    angle = position.double()[:, None, None] * frequencies
    c, s = angle.cos(), angle.sin()
    out = t.clone()
    x, y = (t[..., 0:2 * n:2], t[..., 1:2 * n:2]) if interleaved else (t[..., :n], t[..., n:2 * n])
    u, v = x * c - y * s, x * s + y * c
    if interleaved:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = u, v
    else:
        out[..., :n], out[..., n:2 * n] = u, v
    return out


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,pairs", [(6, 6, 64, 32), (8, 2, 128, 64), (8, 1, 256, 128), (4, 4, 80, 16), (6, 2, 33, 16),
                                                (2, 1, 64, 0), (3, 3, 7, 2), (40, 8, 128, 33)])
def test_append(heads, kv, dim, pairs, dtype, eight):
    gen = torch.Generator().manual_seed(dim + pairs)
    for interleaved in (False, True):
        lengths, new = [1, 40, 33, 17, 0, 900000], [1, 40, 2, 1, 0, 3]
        cache, table, L, starts, q, k, v = make(gen, [1, 40, 33, 17, 0, 20], new, heads, kv, dim, 16, dtype, eight=eight, tail=2)
        if not interleaved:  # a position that 32 bits cannot turn: its page is column 56249
            wide = torch.full((6, 900000 // 16), -1, dtype=torch.int32, device=DEV)
            wide[:, :table.shape[1]] = table
            wide[5, -1] = table[5, 0]
            table = wide
            L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        else:
            lengths[5] = 20
        frequencies = kb.rotary_frequencies(pairs) if pairs else None
        names = ["keys", "values"] + (["key_scales", "value_scales"] if eight else [])
        before = {n: getattr(cache, n).clone() for n in names}
        got = kb.cache_append(cache, table, L, k, v, q=q, starts=starts, frequencies=frequencies, interleaved=interleaved)
        position = torch.cat([torch.arange(a - n, a) for a, n in zip(lengths, new)] + [torch.zeros(2)]).long().to(DEV)
        live = sum(new)
        for t, out in ((q, got),):
            ref = rotated(t, position, frequencies, interleaved)[:live]
            off = (out[:live].double() - ref).abs()
            assert (off <= unit(dtype) * ref.abs() + 8 * 2 ** -24 * 8).all()
            assert (out[live:] == 0).all()
        # what is stored, and that nothing else changed
        of = torch.repeat_interleave(torch.arange(6), torch.tensor(new)).to(DEV)
        page, slot = table.long()[of, position[:live] // 16], position[:live] % 16
        touched = torch.zeros(cache.pages, 16, dtype=torch.bool, device=DEV)
        touched[page, slot] = True
        for name, t in (("key", rotated(k, position, frequencies, interleaved)[:live]), ("value", v[:live].double())):
            now = getattr(cache, name + "s")
            if eight:
                scale = getattr(cache, name + "_scales")[page, :, slot].double()
                want = (t.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
                assert ((scale - want).abs() <= 16 * 2 ** -24 * want + 1e-7 / 448).all()
                back = now.view(torch.uint8)[page, :, slot].view(F8).double() * scale[..., None]
                assert ((back - t).abs() <= (2.0 ** -4 + 1e-6) * t.abs() + (2.0 ** -10 + 1e-6) * scale[..., None] + 8 * 2 ** -24 * 8).all()
            else:
                assert ((now[page, :, slot].double() - t).abs() <= unit(dtype) * t.abs() + 8 * 2 ** -24 * 8).all()
        for n in names:
            a, b = (x.view(torch.uint8) if x.dtype == F8 else x for x in (before[n], getattr(cache, n)))
            assert torch.equal(a.transpose(1, 2)[~touched], b.transpose(1, 2)[~touched])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Parts of one projection, batch-last tensors, pools with the tokens of a page outside its heads, slices of one pool for
    many layers."""
    gen = torch.Generator().manual_seed(3)
    lengths, new = [20, 33], [4, 4]
    cache, table, L, _, q, k, v = make(gen, lengths, new, 4, 2, 64, 16, dtype, token_major=True)
    f = kb.rotary_frequencies(32)
    joined = torch.cat([q, k, v], 1)
    first = kb.cache_append(cache, table, L, joined[:, 4:6], joined[:, 6:], q=joined[:, :4], frequencies=f)
    saved = cache.keys.clone(), cache.values.clone()
    last = [t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in (q, k, v)]  # (features, tokens) in memory
    second = kb.cache_append(cache, table, L, last[1], last[2], q=last[0], frequencies=f)
    assert torch.equal(first, second) and torch.equal(saved[0], cache.keys) and torch.equal(saved[1], cache.values)
    ref = attended(first, cache, table, lengths, new)
    check(kb.cache_attention(first, cache, table, L), ref, cache)
    wide = torch.zeros(8, 9, 64, dtype=dtype, device=DEV)
    out = kb.cache_attention(first, cache, table, L, out=wide[:, 2:6])
    check(out, ref, cache)
    assert (wide[:, :2] == 0).all() and (wide[:, 6:] == 0).all()
    layers = torch.stack([torch.stack([cache.keys, cache.values])] * 3, 2)  # (2, pages, layers, heads, page, dim)
    sub = kb.KVCache.of(layers[0][:, 1], layers[1][:, 1])
    check(kb.cache_attention(first, sub, table, L), ref, cache)
    odd = torch.zeros(cache.keys.numel() + 1, dtype=dtype, device=DEV)[1:].view(cache.pages, 2, 16, 64)  # rows on odd elements
    odd.copy_(cache.keys)
    check(kb.cache_attention(first, kb.KVCache.of(odd, cache.values), table, L), ref, cache)
    wider = torch.full((2, 10), -1, dtype=torch.int32, device=DEV)
    wider[:, :table.shape[1]] = table
    check(kb.cache_attention(first, cache, wider[:, :table.shape[1]], L), ref, cache)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_garbage_outside_a_sequence_is_not_read(dtype, eight):
    """NaN and infinities in unused pages, behind the last token and before the window."""
    gen = torch.Generator().manual_seed(9)
    for lengths, new, window in (([50, 7, 100], [1, 1, 1], None), ([50, 64, 100], [1, 1, 1], 20), ([50, 20, 90], [30, 20, 64], None)):
        cache, table, L, starts, q, _, _ = make(gen, lengths, new, 4, 2, 64, 16, dtype, eight=eight)
        ref = attended(q, cache, table, lengths, new, window=window)
        seen = torch.zeros(cache.pages, 16, dtype=torch.bool, device=DEV)
        for s, n in enumerate(lengths):
            at = torch.arange(0 if window is None else max(0, n - new[s] - window + 1), n, device=DEV)
            seen[table.long()[s, at // 16], at % 16] = True
        for t in [cache.keys, cache.values] + ([cache.key_scales, cache.value_scales] if eight else []):
            if t.dtype == F8:
                t.view(torch.uint8).transpose(1, 2)[~seen] = 0x7f
            else:
                t.transpose(1, 2)[~seen] = math.nan
        check(kb.cache_attention(q, cache, table, L, starts=starts, window=window), ref, cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_not_there(dtype):
    gen = torch.Generator().manual_seed(2)
    for new in ([1, 1, 1, 1], [70, 70, 70, 70]):
        lengths = [100, 100, 100, 100]
        cache, table, L, starts, q, k, v = make(gen, lengths, new, 4, 2, 64, 16, dtype)
        good = attended(q, cache, table, lengths, new)
        table[1, 2] = -1
        table[2, 0] = cache.pages
        L[3] = 16 * table.shape[1] + 1
        out = kb.cache_attention(q, cache, table, L, starts=starts)
        n = new[0]
        check(out[:n], good[:n], cache)
        if n == 1:
            assert torch.isnan(out[n:]).all()
        else:
            # rows of the second sequence at positions 30 and 31 end before the missing page
            check(out[n:n + 2], good[n:n + 2], cache)
            assert torch.isnan(out[n + 2:]).all()
        keys = cache.keys.clone()
        table[0, 6] = 2 ** 31 - 1
        kb.cache_append(cache, table[:1], L[:1], k[:n], v[:n])
        changed = (cache.keys != keys).any(-1).any(1)
        want = torch.zeros_like(changed)
        at = torch.arange(min(100 - n, 96), 96, device=DEV)  # (the last four rows: page 6)
        want[table.long()[0, at // 16], at % 16] = True
        assert torch.equal(changed, want)
        table[0, 6] = -5
        L[:1] = 2 ** 31 - 1
        keys = cache.keys.clone()
        kb.cache_append(cache, table[:1], L[:1], k[:n], v[:n])
        L[:1] = -3
        kb.cache_append(cache, table[:1], L[:1], k[:n], v[:n])
        assert torch.equal(keys, cache.keys)
        assert (kb.cache_attention(q[:n], cache, table[:1], L[:1]) == 0).all()
    kb.check_device()


def test_starts_that_make_no_sense():
    """Starts that fall, or point outside the rows, read and write within the tensors."""
    gen = torch.Generator().manual_seed(2)
    cache, table, L, _, q, k, v = make(gen, [40, 40, 40], [4, 4, 4], 4, 2, 64, 16, torch.float16)
    for starts in ([0, 8, 4, 12], [5, 3, 1, 0], [-7, 2 ** 31 - 1, -2 ** 31, 99], [12, 12, 12, 12], [3, 5, 9, 10]):
        st = torch.tensor(starts, dtype=torch.int32, device=DEV)
        kb.cache_attention(q, cache, table, L, starts=st)
        kb.cache_append(cache, table, L, k, v, q=q, starts=st)
    st = torch.tensor([3, 5, 9, 10], dtype=torch.int32, device=DEV)
    out = kb.cache_attention(q, cache, table, L, starts=st)
    assert (out[:3] == 0).all() and (out[10:] == 0).all() and (out[3:10] != 0).any(-1).all()
    kb.check_device()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_streams_graphs_and_repeats(dtype):
    gen = torch.Generator().manual_seed(8)
    lengths, new = [3000, 1, 700, 64], [1] * 4
    cache, table, L, _, q, k, v = make(gen, lengths, new, 8, 2, 128, 16, dtype)
    ref = kb.cache_attention(q, cache, table, L)
    for _ in range(3):
        assert torch.equal(ref, kb.cache_attention(q, cache, table, L))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(kb.cache_attention(q, cache, table, L))
    torch.cuda.synchronize()
    assert all(torch.equal(ref, o) for o in outs)
    # a step as a graph: the lengths move on between replays
    frequencies = kb.rotary_frequencies(64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rq = kb.cache_append(cache, table, L, k, v, q=q, frequencies=frequencies)
        out = kb.cache_attention(rq, cache, table, L)
    for step in range(3):
        now = [n - step for n in lengths]
        L.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        here = rq.clone()
        torch.cuda.synchronize()
        if step < 1:
            check(out, attended(here, cache, table, now, new), cache)
        else:
            check(out[0::2], attended(here, cache, table, [max(n, 0) for n in now], new)[0::2], cache)
    kb.check_device()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sequences,length", [(1, 1), (1, 512), (1, 513), (2, 4000), (700, 130), (1500, 3)])
def test_few_and_many_sequences(sequences, length, dtype):
    """Whole items, items cut into parts, more sequences than a block has threads; bounds of max_new that do not hold."""
    gen = torch.Generator().manual_seed(sequences + length)
    lengths = [length - s % 2 * (length // 3) for s in range(sequences)]
    cache, table, L, _, q, _, _ = make(gen, lengths, [1] * sequences, 4, 2, 64, 16, dtype)
    check(kb.cache_attention(q, cache, table, L), attended(q, cache, table, lengths, [1] * sequences), cache)
    if sequences <= 2 and length > 600:
        new = [9, 70][:sequences]
        cache, table, L, starts, q, _, _ = make(gen, lengths, new, 4, 2, 64, 16, dtype)
        for bound in (1, 3, None):
            check(kb.cache_attention(q, cache, table, L, starts=starts, max_new=bound), attended(q, cache, table, lengths, new), cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [96, 130, 200])
def test_many_heads_of_one_key_head(heads, dtype):
    gen = torch.Generator().manual_seed(heads)
    for lengths, new in (([1500, 40], [1, 1]), ([300, 90], [2, 60])):
        cache, table, L, starts, q, _, _ = make(gen, lengths, new, heads, 1, 64, 16, dtype)
        check(kb.cache_attention(q, cache, table, L, starts=starts), attended(q, cache, table, lengths, new), cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_tables_and_an_empty_pool(dtype):
    gen = torch.Generator().manual_seed(4)
    cache, table, L, _, q, _, _ = make(gen, [200], [1], 4, 2, 64, 16, dtype)
    q = torch.randn(3, 4, 64, generator=gen).to(dtype).to(DEV)
    L = torch.tensor([200, 150, 7], dtype=torch.int32, device=DEV)
    out = kb.cache_attention(q, cache, table.expand(3, -1), L)  # one prefix, three sequences
    check(out, attended(q, cache, table.expand(3, -1), [200, 150, 7], [1] * 3), cache)
    every = torch.tensor([200, 0, 150, 0, 7, 0], dtype=torch.int32, device=DEV)[::2]  # lengths side by side with something else
    assert torch.equal(out, kb.cache_attention(q, cache, table.expand(3, -1), every))
    none = kb.KVCache.of(cache.keys[:0], cache.values[:0])
    L[2] = 0
    for x, n in ((q, 1), (torch.cat([q] * 90), 90)):
        out = kb.cache_attention(x, none, table.expand(3, -1), L)
        k = torch.zeros(x.shape[0], 2, 64, dtype=dtype, device=DEV)
        kb.cache_append(none, table.expand(3, -1), L, k, k)
        assert torch.isnan(out[:2 * n]).all() and (out[2 * n:] == 0).all()
    with pytest.raises(TypeError):
        kb.cache_attention(q, cache, table.expand(3, -1), L, window=0.5)
    kb.check_device()


def test_empty_calls():
    cache = kb.KVCache(2, 16, 2, 64)
    empty = torch.zeros(0, 2, 64, dtype=torch.float16, device=DEV)
    L, table = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, 1, dtype=torch.int32, device=DEV)
    assert kb.cache_attention(empty, cache, table, L).shape == (0, 2, 64)
    assert kb.cache_append(cache, table, L, empty, empty, q=empty).shape == (0, 2, 64)
    assert kb.cache_append(cache, table[:0], L[:0], empty, empty) is None
    one = torch.ones(3, 2, 64, dtype=torch.float16, device=DEV)
    assert (kb.cache_attention(one, cache, table, L) == 0).all()
    wide = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    assert (kb.cache_attention(one, cache, wide, L) == 0).all()


def test_large_offsets():
    """Pages beyond 2^31 elements of the pool."""
    pages, page, kv, dim = 2 ** 31 // (64 * 128) + 40, 64, 1, 128
    cache = kb.KVCache(pages, page, kv, dim, dtype=torch.bfloat16)
    gen = torch.Generator().manual_seed(1)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=DEV)
    L = torch.tensor([150], dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(150, h, dim, generator=gen).to(torch.bfloat16).to(DEV) for h in (4, 1, 1))
    kb.cache_append(cache, table, L, k, v)
    assert torch.equal(cache.keys[pages - 1, 0], k[:64, 0]) and torch.equal(cache.values[pages - 2, 0, :22], v[128:, 0])
    check(kb.cache_attention(q, cache, table, L), attended(q, cache, table, [150], [150]), cache)
    check(kb.cache_attention(q[-1:], cache, table, L), attended(q[-1:], cache, table, [150], [1]), cache)
