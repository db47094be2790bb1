"""The serving operators of the decoder stack on one GPU: their cases, plain forms and exact values.

A case is a dict of plain values.  ``listed()`` names the fixed ones, ``draw(rng)`` makes another of the same ranges,
``prepare(case, seed)`` builds what a program holds before the call, ``run(state)`` is one pass and returns its outputs,
``work(case)`` the bytes and operations that one pass cannot do without, and ``exact(case, seed)`` what ``run`` returns for
these inputs, in 64 bits.  Where ``own`` is false, ``run`` computes the operators from elementary torch operations.

Operators:

``window``   causal self-attention of whole sequences in which a query sees the last ``window`` keys and the first ``sinks``
             keys of its sequence; grouped heads; any length (``attention_window_fwd``).
``decode``   attention of one new token per sequence over a paged key-value cache, with the same windows (``paged_attention``).
``rope``     norms of queries and keys per head, position rotation, and the new keys' and values' way into the paged cache,
             in one pass over the projection's output (``qk_norm_rope``).
``reserve``  pages taken for the new tokens of every request: block table, slots, positions, lengths (``reserve_slots``).
"""
import functools
import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEAD = 128            # head dimension of the decoder


def listed():
    return [
        # Prefill of two long prompts through a layer with windows, eight key heads for 32 query heads.
        {"name": "window_8192", "op": "window", "batch": 2, "seq": 8192, "heads": 32, "kv_heads": 8, "window": 1024, "sinks": 4,
         "dtype": "bf16"},
        # Prompts whose length is no multiple of any tile, as many key heads as query heads, half precision.
        {"name": "window_ragged_fp16", "op": "window", "batch": 3, "seq": 1000, "heads": 10, "kv_heads": 10, "window": 300,
         "sinks": 1, "dtype": "fp16"},
        # One short prompt on one rank of many: a single key head, no first tokens.
        {"name": "window_short", "op": "window", "batch": 1, "seq": 77, "heads": 4, "kv_heads": 1, "window": 33, "sinks": 0,
         "dtype": "bf16"},
        # The first steps of a single conversation: the smallest call of a decode loop.
        {"name": "decode_one", "op": "decode", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "max_len": 400, "page": 16,
         "order": "page_head", "window": 0, "sinks": 0, "dtype": "bf16"},
        # A serving batch of sequences of all lengths.
        {"name": "decode_64", "op": "decode", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "max_len": 4096, "page": 64,
         "order": "page_slot", "window": 0, "sinks": 0, "dtype": "bf16"},
        # Two very long contexts on a rank that holds a single key head.
        {"name": "decode_long", "op": "decode", "batch": 2, "heads": 8, "kv_heads": 1, "dim": 128, "max_len": 131072, "page": 64,
         "order": "page_slot", "window": 0, "sinks": 0, "dtype": "bf16"},
        # A large batch with windows, 32 key heads of 64, half precision.
        {"name": "decode_window_fp16", "op": "decode", "batch": 256, "heads": 32, "kv_heads": 32, "dim": 64, "max_len": 2048,
         "page": 16, "order": "page_slot", "window": 512, "sinks": 4, "dtype": "fp16"},
        # The prefill of the decoder's default configuration: 16384 tokens, 32 heads.
        {"name": "rope_16384", "op": "rope", "tokens": 16384, "heads": 32, "kv_heads": 32, "dim": 128, "rotary": 128, "norm": True,
         "interleaved": False, "queries_only": False, "page": 64, "order": "page_slot", "theta": 10000.0, "factor": 1.0,
         "dtype": "bf16"},
        # A decode step of 64 sequences far into their contexts: queries out, keys and values only into the cache.
        {"name": "rope_64_decode", "op": "rope", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "norm": True,
         "interleaved": False, "queries_only": True, "page": 16, "order": "page_head", "theta": 500000.0, "factor": 8.0,
         "dtype": "bf16"},
        # A third of every head rotated, pairs side by side, no norms, a head dimension that is no power of two.
        {"name": "rope_part_fp16", "op": "rope", "tokens": 1001, "heads": 12, "kv_heads": 4, "dim": 96, "rotary": 32,
         "norm": False, "interleaved": True, "queries_only": False, "page": 16, "order": "page_slot", "theta": 10000.0,
         "factor": 4.0, "dtype": "fp16"},
        # A decode step of 512 requests: one token each, about one in 16 of them needs a page.
        {"name": "reserve_512_decode", "op": "reserve", "batch": 512, "page": 16, "max_len": 4096, "new": 1, "row_stride": 1,
         "short": False},
        # Prompts of up to 2048 tokens for 32 requests, packed one behind the other, pages running out before the last.
        {"name": "reserve_32_prefill", "op": "reserve", "batch": 32, "page": 64, "max_len": 8192, "new": 2048, "row_stride": 0,
         "short": True},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("window", "decode", "rope", "reserve"))
    dtype = rng.choice(("bf16", "fp16"))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 5, 8))
    if op == "window":
        seq = _between(rng, 1, 7800)
        batch = max(1, min(_between(rng, 1, 16), 60 * 8192 ** 2 // (heads * seq ** 2)))
        return {"op": op, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads,
                "window": _between(rng, 1, min(1024, seq)), "sinks": rng.choice((0, 0, 1, 4, 37)), "dtype": dtype}
    if op == "decode":
        kv_heads = rng.choice((1, 2, 4, 8, 32))
        heads = kv_heads * (rng.choice((1, 2)) if kv_heads == 32 else rng.choice((1, 3, 4, 8, 16)))
        dim = rng.choice((64, 128, 256))
        max_len = _between(rng, 1, min(65536, (1 << 28) // (kv_heads * dim)))
        batch = min(_between(rng, 1, 128), max(1, (1 << 28) // (max_len * kv_heads * dim)))
        return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "max_len": max_len,
                "page": rng.choice((8, 16, 32, 64, 128)), "order": rng.choice(("page_slot", "page_head")),
                "window": rng.choice((0, 0, _between(rng, 1, max_len))), "sinks": rng.choice((0, 4, 37)), "dtype": dtype}
    if op == "rope":
        dim = rng.choice((64, 96, 128, 256))
        rotary = rng.choice((dim, dim, 32, dim // 2))
        return {"op": op, "tokens": _between(rng, 1, 16384), "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
                "norm": rng.random() < 0.7, "interleaved": rng.random() < 0.4, "queries_only": rng.random() < 0.4,
                "page": rng.choice((16, 32, 64)), "order": rng.choice(("page_slot", "page_head")), "theta": 10000.0,
                "factor": rng.choice((1.0, 4.0)), "dtype": dtype}
    batch = _between(rng, 1, 2048)
    prefill = rng.random() < 0.5
    most = max(2, min(2048, 65536 // batch)) if prefill else 1
    return {"op": op, "batch": batch, "page": rng.choice((1, 16, 64, 128)), "max_len": rng.choice((500, 4096, 8192)) + most,
            "new": most, "row_stride": rng.choice((0, most)), "short": rng.random() < 0.3}


# ---- what the cases fix apart from the values: lengths of a decode batch --------------------------------------------

@functools.lru_cache(maxsize=None)
def _decode_lens(batch, max_len):
    """Lengths of a batch: the longest, one of a single token, some that have ended (0), the others in between."""
    rng = random.Random(batch * 1000003 + max_len)
    lens = [rng.randint(max(1, max_len // 8), max_len) for _ in range(batch)]
    lens[batch // 2] = max_len
    if batch > 4:
        lens[0] = 1
        lens[-1] = 0
    return lens


def _visible(n, window, sinks):
    """How many of n keys the newest token sees."""
    start = max(0, n - window) if window else 0
    return min(sinks, start) + n - start


def _cache(case, pages, gen):
    """A layer's pages [pages, page, kv_heads, dim] of keys and of values, in one of two orders in memory: slot before head,
    or head before slot."""
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    both = torch.randn((2, pages, page, kv, dim) if case["order"] == "page_slot" else (2, pages, kv, page, dim), generator=gen,
                       device="cuda", dtype=DTYPES[case["dtype"]])
    if case["order"] == "page_head":
        both = both.transpose(2, 3)
    return both[0], both[1]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "window":
        rows, width = case["batch"] * case["seq"], (case["heads"] + 2 * case["kv_heads"]) * HEAD
        dt = DTYPES[case["dtype"]]
        qkv = torch.randn((rows, width), generator=gen, device="cuda", dtype=dt)
        return {**case, "qkv": qkv, "out": torch.empty((rows, case["heads"] * HEAD), device="cuda", dtype=dt)}
    if op == "decode":
        batch, page, dt = case["batch"], case["page"], DTYPES[case["dtype"]]
        lens = _decode_lens(batch, case["max_len"])
        wide = -(-case["max_len"] // page)
        pages = sum(-(-n // page) for n in lens) + 3
        k, v = _cache(case, pages, gen)
        # pages were handed out in no order, entries behind a sequence's last page were never written
        ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        need = torch.tensor([-(-n // page) for n in lens], device="cuda")
        cols = torch.arange(wide, device="cuda")
        at = (torch.cumsum(need, 0) - need)[:, None] + cols
        table = torch.where(cols < need[:, None], ids[at.clamp(max=pages - 1)], -1).to(torch.int32)
        # queries are the first columns of a projection's output
        both = torch.randn((batch, case["heads"] + 2 * case["kv_heads"], case["dim"]), generator=gen, device="cuda", dtype=dt)
        return {**case, "q": both[:, :case["heads"]], "k": k, "v": v, "table": table,
                "lens": torch.tensor(lens, device="cuda", dtype=torch.int32),
                "out": torch.empty((batch, case["heads"], case["dim"]), device="cuda", dtype=dt),
                "lse": torch.empty((batch, case["heads"]), device="cuda", dtype=torch.float32)}
    if op == "rope":
        tokens, heads, kv, dim, dt = case["tokens"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        qkv = torch.randn((tokens, (heads + 2 * kv) * dim), generator=gen, device="cuda", dtype=dt)
        pages = -(-tokens // case["page"]) + 2
        k, v = (t.zero_() for t in _cache(case, pages, gen))
        state = {**case, "qkv": qkv, "k": k, "v": v, "q_weight": None, "k_weight": None}
        if case["norm"]:
            for name in ("q_weight", "k_weight"):
                state[name] = (1 + 0.1 * torch.randn(dim, generator=gen, device="cuda")).to(dt)
        # a prefill's tokens follow each other; those of a decode step are anywhere
        far = 32768
        if case["queries_only"]:
            state["positions"] = torch.randint(0, far, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
        else:
            first = int(torch.randint(0, far - 16384, (1,), generator=gen, device="cuda"))
            state["positions"] = (first + torch.arange(tokens, device="cuda")).to(torch.int32)
        order = torch.randperm(pages, generator=gen, device="cuda")[:-(-tokens // case["page"])]
        slots = order[:, None] * case["page"] + torch.arange(case["page"], device="cuda")
        state["slots"] = slots.reshape(-1)[:tokens].to(torch.int32)
        angle = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * _speeds(case)
        state["rotation"] = torch.cat([angle.cos(), angle.sin()], 1).to(torch.float32)
        state["out"] = torch.empty((tokens, (heads if case["queries_only"] else heads + 2 * kv) * dim), device="cuda", dtype=dt)
        return state
    batch, page, most = case["batch"], case["page"], case["new"]
    lens = torch.randint(0, case["max_len"] - most + 1, (batch,), generator=gen, device="cuda")
    new = torch.ones_like(lens) if most == 1 else torch.randint(0, most + 1, (batch,), generator=gen, device="cuda")
    if batch > 4:
        new[batch // 3] = 0
    wide = -(-case["max_len"] // page)
    held = (lens + page - 1) // page
    need = int(((lens + new + page - 1) // page - held).sum())
    count = max(1, need * 9 // 10) if case["short"] else need + 7
    pages = batch * wide + count
    ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.where(torch.arange(wide, device="cuda") < held[:, None], ids[count:].view(batch, wide), -1).to(torch.int32)
    tokens = batch * most
    ints = functools.partial(torch.empty, device="cuda", dtype=torch.int32)
    return {**case, "lens": lens.to(torch.int32), "new_lens": new.to(torch.int32), "table": table, "free": ids[:count].clone(),
            "count": torch.tensor([count], device="cuda", dtype=torch.int32), "slots": ints(tokens), "positions": ints(tokens),
            "lens_out": ints(batch), "count_out": ints(1)}


def _speeds(case):
    """Angle per position of every rotated pair, linearly scaled positions."""
    half = case["rotary"] // 2
    return case["theta"] ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half) / case["factor"]


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _FRAMEWORK[state["op"]](state)
    return _PLAIN[state["op"]](state)


@functools.lru_cache(maxsize=None)
def _ops(name):
    return importlib.import_module("iris_b200.ops." + name)


def _own_window(s):
    return _ops("attention").attention_window_fwd(s["qkv"], s["out"], s["batch"], s["seq"], s["heads"], s["kv_heads"],
                                                  window=s["window"], sinks=s["sinks"])


def _own_decode(s):
    _ops("paged").paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["out"], window=s["window"], sinks=s["sinks"],
                                  lse=s["lse"])
    return s["out"], s["lse"]


def _own_rope(s):
    _ops("rotary").qk_norm_rope(s["qkv"], s["out"], s["positions"], s["rotation"], s["heads"], s["kv_heads"], s["dim"],
                                q_weight=s["q_weight"], k_weight=s["k_weight"], interleaved=s["interleaved"], k_cache=s["k"],
                                v_cache=s["v"], slots=s["slots"])
    return s["out"], s["k"], s["v"]


def _own_reserve(s):
    _ops("paged").reserve_slots(s["lens"], s["new_lens"], s["table"], s["free"], s["count"], s["page"], s["slots"],
                                s["positions"], row_stride=s["row_stride"], lens_out=s["lens_out"],
                                free_count_out=s["count_out"])
    return s["slots"], s["positions"], s["table"], s["lens_out"], s["count_out"]


_FRAMEWORK = {"window": _own_window, "decode": _own_decode, "rope": _own_rope, "reserve": _own_reserve}


def _plain_window(s):
    batch, seq, heads, kv = s["batch"], s["seq"], s["heads"], s["kv_heads"]
    x = s["qkv"].view(batch, seq, heads + 2 * kv, HEAD).transpose(1, 2).float()
    q = x[:, :heads].reshape(batch, kv, heads // kv * seq, HEAD)
    k, v = x[:, heads:heads + kv], x[:, heads + kv:]
    i, j = torch.arange(seq, device="cuda")[:, None], torch.arange(seq, device="cuda")
    hidden = (j > i) | ((j <= i - s["window"]) & (j >= s["sinks"]))
    w = torch.matmul(q, k.transpose(2, 3)).view(batch, heads, seq, seq).mul_(HEAD ** -0.5).masked_fill_(hidden, -math.inf)
    w = w.sub_(w.amax(3, keepdim=True)).exp_()
    total = w.sum(3, keepdim=True)
    o = torch.matmul(w.view(batch, kv, -1, seq), v).view(batch, heads, seq, HEAD) / total
    return o.transpose(1, 2).reshape(batch * seq, heads * HEAD).to(s["qkv"].dtype)


def _plain_decode(s):
    q, page, lens = s["q"].float(), s["page"], s["lens"].long()
    batch, heads, dim = q.shape
    kv = s["kv_heads"]
    j = torch.arange(s["max_len"], device="cuda")
    ids = s["table"].long()[:, j // page].clamp(min=0)
    k, v = (t[ids, (j % page).expand_as(ids)].transpose(1, 2).float() for t in (s["k"], s["v"]))   # [batch, kv, max_len, dim]
    seen = j < lens[:, None]
    if s["window"]:
        seen &= (j >= lens[:, None] - s["window"]) | (j < s["sinks"])
    w = torch.matmul(q.view(batch, kv, heads // kv, dim), k.transpose(2, 3)).mul_(dim ** -0.5)
    w = w.masked_fill_(~seen[:, None, None], -math.inf)
    most = w.amax(3, keepdim=True)
    w = w.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = w.sum(3, keepdim=True)
    o = torch.matmul(w, v) / torch.where(total == 0, 1.0, total)
    return o.view(batch, heads, dim).to(s["q"].dtype), (most + total.log()).view(batch, heads)


def _plain_rope(s):
    tokens, heads, kv, dim, half = s["tokens"], s["heads"], s["kv_heads"], s["dim"], s["rotary"] // 2
    x = s["qkv"].view(tokens, heads + 2 * kv, dim)
    turn = s["rotation"][s["positions"].long()]
    cos, sin = turn[:, None, :half], turn[:, None, half:]
    q, k = x[:, :heads].float(), x[:, heads:heads + kv].float()
    if s["norm"]:
        q = q * torch.rsqrt(q.square().mean(2, keepdim=True) + 1e-6) * s["q_weight"].float()
        k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + 1e-6) * s["k_weight"].float()
    x = torch.cat([_turned(q, cos, sin, half, s["interleaved"]), _turned(k, cos, sin, half, s["interleaved"])],
                  1).to(x.dtype), x[:, heads + kv:]
    at, inside = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    s["k"][at, inside] = x[0][:, heads:]
    s["v"][at, inside] = x[1]
    out = x[0][:, :heads] if s["queries_only"] else torch.cat(x, 1)
    return out.reshape(tokens, -1), s["k"], s["v"]


def _turned(x, cos, sin, half, interleaved):
    if interleaved:
        a, b = x[..., :2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], 3).flatten(2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    return torch.cat([y, x[..., 2 * half:]], 2)


def _plain_reserve(s):
    lens, new, page, count = s["lens"].long(), s["new_lens"].long(), s["page"], s["count"].long()
    wide = s["table"].shape[1]
    held = (lens + page - 1) // page
    fits = lens + new <= wide * page
    need = torch.where(fits, (lens + new + page - 1) // page - held, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= count))       # in order, until the free pages run out
    cols = torch.arange(wide, device="cuda")
    fresh = granted[:, None] & (cols >= held[:, None]) & (cols < (held + need)[:, None])
    top = count - 1 - ((upto - need - held)[:, None] + cols)
    s["table"].copy_(torch.where(fresh, s["free"][top.clamp(0, s["free"].numel() - 1)], s["table"]))
    t = torch.arange(s["slots"].numel(), device="cuda")
    ends = torch.cumsum(new, 0)
    if s["row_stride"]:
        req, j = t // s["row_stride"], t % s["row_stride"]
    else:
        req = torch.searchsorted(ends, t, right=True).clamp(max=lens.numel() - 1)
        j = t - (ends - new)[req]
    valid = granted[req] & (j < new[req])
    pos = lens[req] + j
    slot = s["table"][req, (pos // page).clamp(max=wide - 1)].long() * page + pos % page
    used = torch.where(granted & (need > 0), upto, 0).amax()
    return (torch.where(valid, slot, -1).to(torch.int32), torch.where(valid, pos, -1).to(torch.int32), s["table"],
            torch.where(granted, lens + new, lens).to(torch.int32), (count - used).to(torch.int32))


_PLAIN = {"window": _plain_window, "decode": _plain_decode, "rope": _plain_rope, "reserve": _plain_reserve}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "window":
        seq, heads, kv = case["seq"], case["heads"], case["kv_heads"]
        pairs = sum(_visible(i + 1, case["window"], case["sinks"]) for i in range(seq)) * case["batch"] * heads
        return {"bytes": case["batch"] * seq * (2 * heads + 2 * kv) * HEAD * 2, "flops": 4 * HEAD * pairs}
    if op == "decode":
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        keys = sum(_visible(n, case["window"], case["sinks"]) for n in _decode_lens(case["batch"], case["max_len"]))
        return {"bytes": keys * kv * dim * 4 + case["batch"] * heads * (dim * 4 + 4) + case["batch"] * 4 + keys // case["page"] * 4,
                "flops": 4 * dim * heads * keys}
    if op == "rope":
        tokens, heads, kv, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        out = heads if case["queries_only"] else heads + 2 * kv
        return {"bytes": tokens * ((heads + 2 * kv + out + 2 * kv) * dim * 2 + case["rotary"] * 4 + 8),
                "flops": tokens * (heads + kv) * (4 * dim * case["norm"] + 3 * case["rotary"])}
    tokens = case["batch"] * case["new"]
    return {"bytes": tokens * 8 + case["batch"] * 12 + tokens // (2 * case["page"]) * 8, "flops": 0}


# ---- 64 bits, from the definitions -----------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "reserve":
        return None                                          # whole numbers
    s = prepare(case, seed)
    return {"window": _exact_window, "decode": _exact_decode, "rope": _exact_rope}[case["op"]](s)


def _attend(q, k, v):
    """softmax(q . k / sqrt(d)) . v and the logarithm of the softmax's sum, 64 bits; q [n, d], k and v [m, d]."""
    score = torch.einsum("nd,md->nm", q, k) / math.sqrt(q.shape[1])
    return torch.einsum("nm,md->nd", torch.softmax(score, 1), v), torch.logsumexp(score, 1)


def _exact_window(s):
    seq, heads, group = s["seq"], s["heads"], s["heads"] // s["kv_heads"]
    x = s["qkv"].view(s["batch"], seq, heads + 2 * s["kv_heads"], HEAD)
    out = torch.empty((s["batch"], seq, heads, HEAD), dtype=torch.float64, device="cuda")
    at = torch.arange(seq, device="cuda")
    back = at[:, None] - at[None, :]                         # how far a key lies behind a query
    seen = (back >= 0) & ((back < s["window"]) | (at < s["sinks"])[None, :])
    for b in range(s["batch"]):
        for h in range(heads):
            q, k, v = (x[b, :, n].double() for n in (h, heads + h // group, heads + s["kv_heads"] + h // group))
            score = (q @ k.T) / math.sqrt(HEAD)
            out[b, :, h] = torch.softmax(torch.where(seen, score, -math.inf), 1) @ v
    return out.view(s["batch"] * seq, heads * HEAD)


def _exact_decode(s):
    group = s["heads"] // s["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_decode_lens(s["batch"], s["max_len"])):
        start = max(0, n - s["window"]) if s["window"] else 0
        keys = torch.cat([torch.arange(min(s["sinks"], start)), torch.arange(start, n)]).cuda()
        if not len(keys):
            continue
        where = s["table"][b, keys // s["page"]].long(), keys % s["page"]
        k, v = s["k"][where].double(), s["v"][where].double()
        for h in range(s["kv_heads"]):
            rows = slice(h * group, (h + 1) * group)
            out[b, rows], lse[b, rows] = _attend(s["q"][b, rows].double(), k[:, h], v[:, h])
    return out, lse


def _exact_rope(s):
    heads, kv, dim, rot = s["heads"], s["kv_heads"], s["dim"], s["rotary"]
    x = s["qkv"].view(s["tokens"], -1, dim).double()
    if s["norm"]:
        for part, weight in ((slice(0, heads), "q_weight"), (slice(heads, heads + kv), "k_weight")):
            x[:, part] *= s[weight].double() / torch.sqrt((x[:, part] ** 2).sum(2, keepdim=True) / dim + 1e-6)
    # the pair of components of a rotated plane as one complex number, turned by multiplication
    first = torch.arange(0, rot, 2, device="cuda") if s["interleaved"] else torch.arange(rot // 2, device="cuda")
    second = first + (1 if s["interleaved"] else rot // 2)
    angle = s["positions"].double()[:, None] * _speeds(s)
    turned = torch.complex(x[:, :heads + kv, first], x[:, :heads + kv, second]) * torch.exp(1j * angle)[:, None]
    x[:, :heads + kv, first], x[:, :heads + kv, second] = turned.real, turned.imag
    k, v = s["k"].double(), s["v"].double()
    page, inside = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    k[page, inside], v[page, inside] = x[:, heads:heads + kv], x[:, heads + kv:]
    return (x[:, :heads] if s["queries_only"] else x).reshape(s["tokens"], -1), k, v
