"""The operators of a generating model's attention as measurable cases.

Keys and values of many sequences live in pages of one pool; ``table[s, i]`` is the page that holds tokens
``i * page .. (i + 1) * page - 1`` of sequence ``s``, ``lengths[s]`` its tokens, the new ones included.

* ``append``: the new tokens' queries and keys are rotated by their positions, keys and values stored
  (``cache_append``), in the model's type or in 8 bits with a scale for each token and head;
* ``attend``: attention of the new tokens over their sequence's cache, causal (``cache_attention``): one new token for
  each sequence, a prompt's many, or a batch of both (``new`` = 0).

Where ``own`` is false the operators are elementary torch operations in 32 bits (angles in 64), rounded once at the end.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
F8 = torch.float8_e4m3fn

#          heads, kv_heads, dim
SMALL = (6, 6, 64)
BASE = (12, 12, 64)
WIDE = (32, 8, 128)
OTHERS = ((16, 2, 128), (8, 1, 256), (16, 16, 80), (24, 8, 96), (20, 4, 64), (40, 10, 128))


def _case(name, op, dtype, heads, page, sequences, low, high, new=1, most_new=1, tail=0, eight=False, window=0, interleaved=False):
    return {"name": name, "op": op, "dtype": dtype, "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "page": page,
            "sequences": sequences, "low": low, "high": high, "new": new, "most_new": most_new, "tail": tail, "eight": eight,
            "window": window, "interleaved": interleaved}


def listed():
    return [
        # a handful of sequences answered online: launches and host work are all there is
        _case("append_online_fp16", "append", "fp16", BASE, 16, 8, 1, 500),
        # a serving batch at full load, 8-bit cache
        _case("append_batch_eight", "append", "bf16", WIDE, 64, 256, 1, 4096, eight=True),
        # the prompts of a wide model over long sequences
        _case("append_prompts_bf16", "append", "bf16", WIDE, 64, 4, 8192, 8192, new=8192),
        # the same handful of sequences, attended to
        _case("attend_online_fp16", "attend", "fp16", BASE, 16, 8, 1, 500),
        # a serving batch, sequences of every length
        _case("attend_batch_bf16", "attend", "bf16", WIDE, 64, 64, 1, 8192),
        # one very long document
        _case("attend_long_bf16", "attend", "bf16", WIDE, 16, 1, 131077, 131077),
        # a larger batch in an 8-bit cache
        _case("attend_batch_eight", "attend", "bf16", WIDE, 64, 128, 1, 8192, eight=True),
        # a model with a sliding window and one wide key head
        _case("attend_window_fp16", "attend", "fp16", (8, 1, 256), 32, 96, 1, 16000, window=4096),
        # inference in fp32
        _case("attend_batch_fp32", "attend", "fp32", BASE, 16, 32, 1, 2047),
        # single tokens of some sequences beside chunks of others' prompts, padded to a captured size
        _case("attend_mixed_bf16", "attend", "bf16", WIDE, 16, 24, 1, 4096, new=0, most_new=512, tail=37),
        # a batch of short prompts
        _case("attend_prompts_fp16", "attend", "fp16", BASE, 16, 32, 1000, 1000, new=1000),
        # a long prompt
        _case("attend_prompt_bf16", "attend", "bf16", WIDE, 64, 1, 8192, 8192, new=8192),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend"))
    dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
    heads = rng.choice((SMALL, BASE, WIDE, WIDE) + OTHERS)
    page = rng.choice((16, 16, 32, 64, 128, 256))
    kind = rng.choice(("one", "one", "few", "prompts", "mixed"))
    sequences = _log(rng, 1, 256 if kind in ("one", "few") else 32)
    eight = dtype != "fp32" and rng.random() < 0.3
    window = _log(rng, 64, 8192) if rng.random() < 0.2 else 0
    # a pool of at most 2^28 values, queries and scores that stay below the largest listed case's
    most = max(2, min(131072, (1 << 28) // (2 * sequences * heads[1] * heads[2])))
    case = dict(op=op, dtype=dtype, heads=heads, page=page, sequences=sequences, eight=eight, window=window if op == "attend" else 0)
    if kind in ("one", "few"):
        case.update(high=_log(rng, 1, most), new=1 if kind == "one" else rng.randint(2, 8))
        case["low"] = 1 if rng.random() < 0.7 else case["high"]
    else:
        pairs = min(1 << 31, (1 << 38) // heads[2]) // (heads[0] * sequences) // (4 if dtype == "fp32" else 1)
        high = _log(rng, 16, max(17, min(most, 8192, int(math.sqrt(pairs)))))
        if kind == "prompts":
            case.update(low=high, high=high, new=high)
        else:
            case.update(low=1, high=high, new=0, most_new=rng.randint(1, high), tail=rng.randint(0, 40))
    case["interleaved"] = op == "append" and rng.random() < 0.3
    case = _case("", case.pop("op"), case.pop("dtype"), case.pop("heads"), **case)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# sizes (the case's alone: what is drawn with the seed does not change the work)
# ---------------------------------------------------------------------------
def _sizes(case):
    """The lengths of the sequences and their new tokens."""
    rng = random.Random("%(sequences)d %(low)d %(high)d %(new)d %(most_new)d" % case)
    lengths = [rng.randint(case["low"], case["high"]) for _ in range(case["sequences"])]
    if case["new"]:
        new = [case["new"]] * len(lengths)
        lengths = [max(n, m) for n, m in zip(lengths, new)]
    else:
        new = [1 if rng.random() < 0.5 else rng.randint(1, case["most_new"]) for _ in lengths]
        lengths = [max(n, m) for n, m in zip(lengths, new)]
    return lengths, new


def _tokens(case):
    return sum(_sizes(case)[1]) + case["tail"]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _projected(gen, tokens, heads, dim):
    """What a projection gives: a few features stand out in every head."""
    return _randn(gen, tokens, heads, dim) * (1 + 2 * (torch.rand(heads, dim, device="cuda", generator=gen) > 0.97))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, heads, kv, dim = DTYPES[case["dtype"]], case["page"], case["heads"], case["kv_heads"], case["dim"]
    lengths, new = _sizes(case)
    used = [-(-n // page) for n in lengths]
    # a pool somewhat larger than what is used, pages in no order; entries behind a sequence's last page mean nothing
    pages = sum(used) + 8
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).tolist()
    table = torch.full((len(lengths), max(used)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    tokens = _tokens(case)
    state = {"case": case, "table": table.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
             "longest": max(lengths), "most": max(new), "starts": None, "q": _projected(gen, tokens, heads, dim).to(dtype)}
    if not case["new"]:
        state["starts"] = torch.tensor([sum(new[:s]) for s in range(len(new) + 1)], dtype=torch.int32).cuda()
    if case["op"] == "append":
        # parts of what one grouped projection returns
        both = torch.stack([_projected(gen, tokens, kv, dim), _randn(gen, tokens, kv, dim)]).to(dtype)
        state["k"], state["v"] = both[0], both[1]
        state["frequencies"] = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device="cuda") / (dim // 2))
    keys, values = (f(gen, pages, kv, page, dim) for f in (lambda g, p, h, r, d: _projected(g, p * r, h, d).view(p, r, h, d).transpose(1, 2).contiguous(), _randn))
    state["key_scales"] = state["value_scales"] = None
    if case["eight"]:
        for name, t in (("key", keys), ("value", values)):
            scale = t.abs().amax(-1) / 448
            state[name + "s"] = (t / scale.unsqueeze(-1)).to(F8)
            state[name + "_scales"] = scale
    else:
        state["keys"], state["values"] = keys.to(dtype), values.to(dtype)
    if own:
        import ksmm_b200 as kb

        state["cache"] = kb.KVCache.of(state["keys"], state["values"], state["key_scales"], state["value_scales"])
    return state


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(state):
    import ksmm_b200 as kb

    case, cache, table, lengths, starts = state["case"], state["cache"], state["table"], state["lengths"], state["starts"]
    if case["op"] == "append":
        q = kb.cache_append(cache, table, lengths, state["k"], state["v"], q=state["q"], starts=starts,
                            frequencies=state["frequencies"], interleaved=case["interleaved"])
        return [q, cache.keys, cache.values, cache.key_scales, cache.value_scales]
    return kb.cache_attention(state["q"], cache, table, lengths, starts=starts, window=case["window"] or None)


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _first(state):
    """Where each sequence's new tokens start in the rows of q, (sequences + 1,)."""
    if state["starts"] is not None:
        return state["starts"].long()
    n = state["case"]["new"]
    return torch.arange(0, n * state["case"]["sequences"] + 1, n, device="cuda")


def _rotate(t, angles, interleaved):
    cos, sin = angles.cos().float().unsqueeze(1), angles.sin().float().unsqueeze(1)
    t = t.float()
    if interleaved:
        x, y = t[..., 0::2], t[..., 1::2]
        return torch.stack([x * cos - y * sin, x * sin + y * cos], -1).flatten(-2)
    x, y = t.chunk(2, -1)
    return torch.cat([x * cos - y * sin, x * sin + y * cos], -1)


def _plain_append(state):
    case, dtype, page = state["case"], DTYPES[state["case"]["dtype"]], state["case"]["page"]
    first = _first(state)
    token = torch.arange(state["q"].shape[0], device="cuda")
    of = torch.searchsorted(first, token, right=True) - 1
    there = of < case["sequences"]                      # (rows behind the last sequence belong to none)
    of = of.clamp(max=case["sequences"] - 1)
    position = state["lengths"].long()[of] - first[of + 1] + token
    angles = position.clamp(min=0).double().unsqueeze(1) * state["frequencies"]
    position = torch.where(there, position, 0)
    q = torch.where(there[:, None, None], _rotate(state["q"], angles, case["interleaved"]), 0.0).to(dtype)
    rows = state["q"].shape[0] - case["tail"]
    to = state["table"].long()[of, position // page][:rows], (position % page)[:rows]
    for name, t in (("key", _rotate(state["k"], angles, case["interleaved"])), ("value", state["v"].float())):
        t = t[:rows]
        if case["eight"]:
            scale = (t.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
            state[name + "_scales"][to[0], :, to[1]] = scale
            state[name + "s"].view(torch.uint8)[to[0], :, to[1]] = (t / scale.unsqueeze(-1)).to(F8).view(torch.uint8)
        else:
            state[name + "s"][to[0], :, to[1]] = t.to(dtype)
    return [q, state["keys"], state["values"], state["key_scales"], state["value_scales"]]


def _gathered(state, name, at, page):
    t = state[name + "s"]
    t = (t.view(torch.uint8)[page, :, at].view(F8) if t.dtype == F8 else t[page, :, at]).float()
    scales = state[name + "_scales"]
    return (t if scales is None else t * scales[page, :, at].unsqueeze(-1)).transpose(1, 2)  # (S, kv_heads, longest, dim)


def _plain_attend(state):
    case, q, dtype = state["case"], state["q"], DTYPES[state["case"]["dtype"]]
    S, kv, dim, most, longest = case["sequences"], case["kv_heads"], case["dim"], state["most"], state["longest"]
    group = case["heads"] // kv
    first, lengths = _first(state), state["lengths"].long()
    new = first[1:] - first[:-1]
    k_at = torch.arange(longest, device="cuda")
    page = state["table"].long()[:, k_at // case["page"]].clamp(min=0)
    keys, values = (_gathered(state, name, k_at % case["page"], page) for name in ("key", "value"))
    nth = torch.arange(most, device="cuda")
    row = first[:-1, None] + nth                                                             # (S, most)
    there = nth < new[:, None]
    rows = q[row.clamp(max=q.shape[0] - 1)].float().view(S, most, kv, group, dim).permute(0, 2, 3, 1, 4)
    scores = (rows.reshape(S, kv, group * most, dim) @ keys.transpose(-1, -2)).view(S, kv, group, most, longest) / math.sqrt(dim)
    q_at = (lengths - new)[:, None] + nth
    seen = (k_at <= q_at[..., None]) & there[..., None]
    if case["window"]:
        seen &= k_at > q_at[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = weights.sum(-1, keepdim=True)
    o = (weights.view(S, kv, group * most, longest) @ values).view(S, kv, group, most, dim) / torch.where(total == 0, 1.0, total)
    out = torch.zeros(q.shape[0] + 1, *q.shape[1:], device="cuda")
    out[torch.where(there, row, q.shape[0])] = o.permute(0, 3, 1, 2, 4).reshape(S, most, kv * group, dim)
    return out[:-1].to(dtype)


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attend(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    lengths, new = _sizes(case)
    es, kv, heads, dim = ESIZE[case["dtype"]], case["kv_heads"], case["heads"], case["dim"]
    row = dim + 4 if case["eight"] else dim * es                     # a token's key of one head in the cache
    tokens = sum(new)
    indexes = 4 * sum(2 - (-n // case["page"]) for n in lengths)
    if case["op"] == "append":
        return {"bytes": tokens * (2 * heads * dim * es + 2 * kv * (dim * es + row)) + indexes, "flops": 3 * tokens * (heads + kv) * dim}
    window, read, pairs = case["window"], 0, 0
    for length, n in zip(lengths, new):
        start = length - n
        read += min(length, window + n - 1) if window else length
        if not window:
            pairs += n * start + n * (n + 1) // 2
        else:
            short = max(0, min(n, window - start))                   # tokens whose window reaches the first key
            pairs += short * start + short * (short + 1) // 2 + (n - short) * window
    return {"bytes": 2 * read * kv * row + 2 * tokens * heads * dim * es + indexes, "flops": 4 * pairs * heads * dim}


# ---------------------------------------------------------------------------
# the definition in 64 bits, a sequence at a time
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    lengths, new = _sizes(case)
    page, group = case["page"], case["heads"] // case["kv_heads"]
    table, q = state["table"].cpu(), state["q"].double()
    pool = {name: (state[name + "s"], state[name + "_scales"]) for name in ("key", "value")}
    out = torch.zeros_like(q)
    made = {name: t.double() for name, (t, _) in pool.items()} if case["op"] == "append" else None
    scales = {name: None if s is None else s.double() for name, (_, s) in pool.items()}
    at = 0
    for s, (length, n) in enumerate(zip(lengths, new)):
        rows = slice(at, at + n)
        at += n
        if case["op"] == "append":
            position = torch.arange(length - n, length, device="cuda")
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), position.double()[:, None] * state["frequencies"])[:, None]

            def turned(t):
                if case["interleaved"]:
                    return torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
                c = torch.complex(*(h.contiguous() for h in t.tensor_split(2, -1))) * turn
                return torch.cat([c.real, c.imag], -1)

            out[rows] = turned(q[rows])
            where = table[s][(position // page).cpu()].long().cuda()
            for name, t in (("key", turned(state["k"][rows].double())), ("value", state["v"][rows].double())):
                if case["eight"]:
                    scale = (t.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
                    scales[name][where, :, position % page] = scale
                    t = (t / scale.float().double()[..., None]).to(F8).double()
                made[name][where, :, position % page] = t
            continue
        used = table[s, :-(-length // page)].long().cuda()
        k, v = (t[used].double() * (1 if sc is None else sc[used].double()[..., None]) for t, sc in (pool["key"], pool["value"]))
        k, v = (t.transpose(0, 1).flatten(1, 2)[:, :length] for t in (k, v))                     # (kv_heads, length, dim)
        q_at, k_at = torch.arange(length - n, length, device="cuda")[:, None], torch.arange(length, device="cuda")
        hidden = (k_at > q_at) | ((k_at <= q_at - case["window"]) if case["window"] else torch.zeros_like(k_at > q_at))
        for h in range(case["heads"]):
            w = torch.softmax((q[rows, h] @ k[h // group].t() / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf), -1)
            out[rows, h] = w @ v[h // group]
    if case["op"] == "append":
        return [out, made["key"], made["value"], scales["key"], scales["value"]]
    return out
