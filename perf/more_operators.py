"""Masked and capped attention over pages, pages held in 4 bits, eviction by weight.

A case is one call (or two that belong together) of one operator on one shape:

  prompt   several new tokens of each sequence attend over its pages: capped scores, a bias
           by distance, a window, documents, prefixes that are seen from both sides
  token    the same for one new token a sequence
  append4  keys and values written into pages of 4-bit values, and read back
  attend4  one new token a sequence over pages of 4-bit values
  step4    a decode step on them: one token appended, its attention, and the row as it is held
  weigh    one new token a sequence, and what its attention gave to each cached token added up
  evict    the tokens of the largest weight, and the newest, moved to other pages

``listed`` holds generic sizes and those of the repository's own configurations, ``draw``
more of the same ranges.  ``run`` computes the operators in elementary torch operations
where ``own`` is false, and through the library where it is true; ``exact`` restates them
in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 32  # channels that share a scale


def _case(kind, **kw):
    c = dict(kind=kind, sequences=1, tokens=1, least=0, new=1, q_heads=8, heads=8, dim=128,
             page_size=16, dtype="bfloat16", rotary=False, base=10000.0, softcap=0.0,
             slopes=False, window=0, prefix=0, document=0, keep=0, recent=0)
    c.update(kw)
    return c


def listed():
    return [
        # draft tokens of a server's sequences, checked in one pass behind what they hold
        _case("prompt", name="prompt_draft", sequences=8, tokens=1500, least=40, new=6,
              q_heads=32, rotary=True, softcap=50.0),
        # documents packed into long rows, each with a prefix that it sees whole, scores biased
        # by distance: a batch of odd lengths behind cached beginnings
        _case("prompt", name="prompt_packed", sequences=5, tokens=300, new=2011, q_heads=14,
              heads=2, dim=64, dtype="float16", slopes=True, prefix=37, document=450),
        # fp32 rows of a head dimension that is no power of two, a window behind a few first
        # tokens that stay seen, capped scores
        _case("prompt", name="prompt_window", sequences=3, tokens=0, new=1277, q_heads=12,
              heads=4, dim=96, page_size=48, dtype="float32", softcap=30.0, window=500, prefix=4),
        # one long prompt: the matrix cores' rate
        _case("prompt", name="prompt_long", tokens=0, new=8192, q_heads=32, page_size=64,
              rotary=True, base=500000.0),
        # a chat's next token, biased by distance: latency alone
        _case("token", name="token_bias", tokens=511, least=511, q_heads=14, heads=14, dim=64,
              dtype="float16", slopes=True),
        # a server's ragged batch with capped scores, a window and first tokens that stay seen
        _case("token", name="token_capped", sequences=32, tokens=8192, least=100, q_heads=32,
              page_size=32, rotary=True, softcap=50.0, window=4096, prefix=16),
        # ragged prompts arriving together
        _case("append4", name="append4_prompts", sequences=16, tokens=640, new=2048, dim=128,
              page_size=64),
        # a chat's decode step
        _case("step4", name="step4_token", tokens=511, least=511, q_heads=14, heads=2, dim=64,
              dtype="float16"),
        # one layer of 64 sequences of 8,192 tokens: the memory's rate
        _case("attend4", name="attend4_batch", sequences=64, tokens=8192, least=8192, q_heads=32,
              page_size=64, rotary=True),
        # a server's batch of sequences whose caches have a budget
        _case("weigh", name="weigh_batch", sequences=24, tokens=4096, least=512, q_heads=32,
              page_size=64),
        # sequences over their budget, halved
        _case("evict", name="evict_batch", sequences=24, tokens=4096, least=1500, page_size=64,
              keep=2048, recent=256),
        # one long chat, most of it dropped
        _case("evict", name="evict_chat", tokens=32768, least=32768, page_size=64, keep=8192,
              recent=1024),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "prompt", "token", "token", "append4", "attend4",
                       "step4", "weigh", "evict"))
    heads = rng.choice((1, 2, 4, 4, 8, 8, 14))
    four = kind.endswith("4")
    dim = rng.choice((64, 96, 128, 128, 256) if four else (64, 64, 80, 96, 128, 128, 128, 256))
    c = dict(heads=heads, dim=dim, dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
             q_heads=heads * rng.choice((1, 2, 3, 4, 4, 7, 8)),
             page_size=rng.choice((16, 16, 32, 48, 64, 128, 256)),
             base=rng.choice((10000.0, 500000.0)))
    if kind in ("prompt", "token", "attend4"):
        c["rotary"] = rng.random() < 0.5
    if kind in ("prompt", "token", "weigh"):
        c["softcap"] = rng.choice((0.0, 0.0, 30.0, 50.0))
        c["slopes"] = rng.random() < 0.3
        c["window"] = rng.choice((0, 0, 0, _spread(rng, 16, 4096)))
        c["prefix"] = rng.choice((0, 0, _spread(rng, 1, 300)))
        c["document"] = rng.choice((0, 0, 0, _spread(rng, 30, 3000)))
    tokens = _spread(rng, 1, 65536)
    sequences = _spread(rng, 1, 128)
    if kind == "prompt":
        new, tokens, sequences = _spread(rng, 1, 8192), _spread(rng, 1, 16384), min(sequences, 32)
        limit = 1 << (30 if c["dtype"] != "float32" else 27)
        while sequences * new * (tokens + new) * c["q_heads"] * dim // 128 > limit or \
                sequences * (tokens + new) * heads * dim > 1 << 26:
            sequences, new = max(1, sequences // 2), max(1, new * 2 // 3)
            tokens = max(1, tokens * 3 // 4)
        return _case(kind, **{**c, "sequences": sequences, "tokens": tokens, "new": new,
                              "least": rng.choice((0, tokens))})
    if kind == "append4":
        tokens, new = _spread(rng, 1, 4096), rng.choice((1, _spread(rng, 2, 40000)))
        while sequences > 1 and sequences * new * heads * dim > 1 << 25:
            sequences //= 2
        while sequences * new * heads * dim > 1 << 25:
            new //= 2
        return _case(kind, **{**c, "sequences": sequences, "tokens": tokens, "new": new,
                              "least": rng.choice((0, tokens))})
    limit = {"attend4": 1 << 28, "step4": 1 << 25}.get(kind, 1 << 27)
    while sequences * tokens * heads * dim * max(1, c["q_heads"] // heads // 4) > limit:
        sequences, tokens = max(1, sequences // 2), max(1, tokens * 3 // 4)
    c["least"] = rng.choice((0, 1, tokens // 4, tokens))
    if kind == "evict":
        c["keep"] = _spread(rng, 1, tokens)
        c["recent"] = rng.choice((0, c["keep"], c["keep"] // 8))
    return _case(kind, **{**c, "sequences": sequences, "tokens": tokens})


# ---------------------------------------------------------------- the shapes

def _counts(c):
    """Per sequence: the tokens it holds before the call, and the new ones."""
    rng = random.Random(c["tokens"] * 1000003 + c["sequences"])
    lengths = [rng.randint(c["least"], c["tokens"]) for _ in range(c["sequences"])]
    lengths[0], lengths[-1] = c["least"], c["tokens"]
    new = [rng.randint(1, c["new"]) for _ in lengths]
    new[0] = c["new"]
    return lengths, new


def _queries(c):
    """Of every query, as tensors: its sequence, position, the tokens there are, the first that
    it may see and the end of what it sees from both sides."""
    lengths, new = _counts(c)
    several = c["kind"] == "prompt"
    owner = torch.tensor([i for i, m in enumerate(new) for _ in range(m if several else 1)])
    if several:
        n = torch.tensor([a + b for a, b in zip(lengths, new)])[owner]
        at = torch.tensor([lengths[i] + j for i, m in enumerate(new) for j in range(m)])
    else:
        n = torch.tensor(lengths)
        at = n - 1
    doc = c["document"]
    first = at.clamp(min=0) // doc * doc if doc else torch.zeros_like(at)
    prefix = torch.minimum(first + c["prefix"], n) if c["prefix"] else torch.zeros_like(at)
    return owner, at, n, first, prefix


def _seen(c):
    """Tokens that each query sees."""
    _, at, n, first, prefix = _queries(c)
    end = torch.minimum(n, torch.maximum(at + 1, prefix))
    seen = (end - first).clamp(min=0)
    if c["window"]:
        hidden = torch.minimum(at - c["window"] + 1, end) - torch.maximum(prefix, first)
        seen -= hidden.clamp(min=0)
    return seen


def work(c):
    size = 4 if c["dtype"] == "float32" else 2
    kind, d, h, hq = c["kind"], c["dim"], c["heads"], c["q_heads"]
    lengths, new = _counts(c)
    held = d // 2 + -(-d // BLOCK)  # bytes of a row in 4 bits
    if kind == "append4":
        rows = 2 * sum(new) * h
        return {"bytes": rows * (d * size + held + held + 4 * d), "flops": 4 * rows * d}
    if kind == "evict":
        moved = sum(min(n, c["keep"]) for n in lengths)
        over = sum(n for n in lengths if n > c["keep"])
        return {"bytes": h * (8 * over + moved * 4 * d * size + 4 * c["keep"] * len(lengths)),
                "flops": h * over}
    if kind in ("attend4", "step4"):
        seen = sum(lengths) + (len(lengths) if kind == "step4" else 0)
        rows = 2 * h * sum(lengths)
        step = len(lengths) * h * 2 * (d * size + held + 4 * d) if kind == "step4" else 0
        return {"bytes": rows * held + 2 * len(lengths) * hq * d * size + step,
                "flops": 4 * seen * hq * d}
    seen = _seen(c)
    pairs = int(seen.sum())
    rows = 2 * h * (int(seen.sum()) if kind != "prompt" else _rows_seen(c))
    io = 2 * len(seen) * hq * d * size
    return {"bytes": rows * d * size + io + (8 * h * pairs if kind == "weigh" else 0),
            "flops": 4 * pairs * hq * d}


def _rows_seen(c):
    """Rows that any query sees, over the sequences."""
    owner, at, n, first, prefix = _queries(c)
    total = 0
    for i in range(c["sequences"]):
        of = owner == i
        a, e = first[of], torch.minimum(n, torch.maximum(at + 1, prefix))[of]
        lo = torch.maximum(a, at[of] - c["window"] + 1) if c["window"] else a
        edge = torch.zeros(int(n[of][0]) + 1, dtype=torch.int64)
        for x, y in ((lo, e), (a, torch.minimum(prefix[of], e))):
            some = y > x
            edge.index_add_(0, x[some], torch.ones_like(x[some]))
            edge.index_add_(0, y[some], -torch.ones_like(y[some]))
        total += int((edge.cumsum(0) > 0).sum())
    return total


# ---------------------------------------------------------------- the inputs

def _tables(c, rng, counts):
    """The pages of sequences of so many tokens among a pool's, anywhere in it."""
    ps = c["page_size"]
    need = [(n + ps - 1) // ps for n in counts]
    pages = sum(need) + 8
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.zeros(len(counts), max(1, max(need)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, pages


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    rng = random.Random(seed)
    kind, ps, h, d = c["kind"], c["page_size"], c["heads"], c["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    lengths, new = _counts(c)
    grows = kind in ("append4", "step4")
    if kind in ("prompt",) or grows:
        counts = [n + m for n, m in zip(lengths, new)]
    else:
        counts = lengths
    total = sum(new)
    if kind == "evict":  # each sequence has pages to move to beside its own
        b = len(lengths)
        table, pages = _tables(c, rng, [*counts, *[c["keep"]] * b])
        s = {"table": table[:b].cuda(),
             "into": table[b:, :(c["keep"] + ps - 1) // ps].contiguous().cuda()}
    else:
        table, pages = _tables(c, rng, counts)
        s = {"table": table.cuda()}
    # where each of the sequences' tokens lies, as a program that places them itself keeps it
    held = counts if kind == "prompt" else lengths
    s["lengths"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    # heads differ in scale, as the keys and values of a model do
    scale = torch.exp(0.5 * torch.randn(2, h, 1, 1, generator=g, device="cuda")).to(dtype)
    if kind in ("attend4", "step4"):  # a cached token's rows, appended before
        n = sum(lengths)
        s["old_k"] = normal(n, h, d).mul_(scale[0, :, :, 0])
        s["old_v"] = normal(n, h, d).mul_(scale[1, :, :, 0])
        s["old_offsets"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)],
                                        dtype=torch.int32, device="cuda")
    elif kind != "append4":
        s["k_pages"] = normal(pages, h, ps, d).mul_(scale[0])
        s["v_pages"] = normal(pages, h, ps, d).mul_(scale[1])
    if kind in ("append4", "step4"):
        s["k"] = normal(total, h, d).mul_(scale[0, :, :, 0])
        s["v"] = normal(total, h, d).mul_(scale[1, :, :, 0])
    s["pages"] = pages
    if kind == "prompt" or kind == "append4":
        s["offsets"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)],
                                    dtype=torch.int32, device="cuda")
    if kind not in ("append4", "evict"):
        s["q"] = normal(total if kind == "prompt" else c["sequences"], c["q_heads"], d)
    if kind in ("weigh", "evict"):
        capacity = table.shape[1] * ps
        weights = torch.rand(c["sequences"], h, capacity, generator=g, device="cuda") ** 8
        if kind == "evict":  # many tokens that nothing looked at: ties
            weights = torch.where(weights < 1e-3, 0.0, weights)
        at = torch.arange(capacity, device="cuda")
        s["weights"] = torch.where(at < s["lengths"][:, None, None], weights, 0.0)
    s["slopes"] = None
    if c["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / c["q_heads"])
                                    for i in range(c["q_heads"])], device="cuda")
    if kind in ("prompt", "token", "weigh"):
        owner, at, n, first, prefix = _queries(c)
        s["owner"], s["at"] = owner.cuda(), at.cuda()
        s["first"] = first.int().cuda() if c["document"] else None
        s["prefix"] = prefix.int().cuda() if c["prefix"] else None
        if kind == "prompt":
            s["place"] = torch.tensor([j for m in new for j in range(m)]).cuda()
    if grows:
        one = kind == "step4"
        s["owner"] = torch.tensor([i for i, m in enumerate(new) for _ in range(1 if one else m)],
                                  device="cuda")
        s["place"] = torch.tensor([lengths[i] + j for i, m in enumerate(new)
                                   for j in range(1 if one else m)], device="cuda")
    return s


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    four = c["kind"] in ("append4", "attend4", "step4")
    if own:
        from adaptq_amd import paged
        from adaptq_amd.rotary import Rotary
        rotary = Rotary(c["dim"], base=c["base"]) if c["rotary"] else None
        if four:
            s["cache"] = paged.PagedCache4.allocate(s["pages"], c["heads"], c["page_size"], c["dim"],
                                                    dtype=DTYPES[c["dtype"]], rotary=rotary)
        else:
            s["cache"] = paged.PagedCache(s["k_pages"], s["v_pages"], rotary=rotary)
    else:
        if c["rotary"]:
            i = torch.arange(c["dim"] // 2, dtype=torch.float64, device="cuda")
            s["frequencies"] = c["base"] ** (-2.0 * i / c["dim"])
        if four:
            shape = (s["pages"], c["heads"], c["page_size"])
            for x in ("k", "v"):
                s[x + "_codes"] = torch.zeros(*shape, c["dim"] // 2, dtype=torch.uint8,
                                              device="cuda")
                s[x + "_scales"] = torch.zeros(*shape, -(-c["dim"] // BLOCK), dtype=torch.uint8,
                                               device="cuda")
    if "old_k" in s:  # what the sequences hold
        k, v, at = s.pop("old_k"), s.pop("old_v"), s.pop("old_offsets")
        if own:
            zero = torch.zeros_like(s["lengths"])
            if c["rotary"]:  # the rows come as they are to lie in the pages
                plain = paged.PagedCache4(s["cache"].k_pages, s["cache"].v_pages,
                                          dtype=DTYPES[c["dtype"]])
                plain.append(k, v, s["table"], zero, offsets=at)
            else:
                s["cache"].append(k, v, s["table"], zero, offsets=at)
        else:
            n = s["lengths"].long()
            owner = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n)
            place = torch.arange(len(owner), device="cuda") - at.long()[owner]
            _put4(s, k, v, owner, place)
    return s


# ---------------------------------------------------------------- the plain forms

def _rotate(s, x, at):
    """x [tokens, heads, dim] at positions [tokens], in 32 bits."""
    x = x.float()
    if not s["case"]["rotary"]:
        return x
    angle = at.double()[:, None] * s["frequencies"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _shaped(s, score, distance, slopes):
    """Scores as they enter the softmax; slopes [heads of the scores], by their last two dims."""
    cap = s["case"]["softcap"]
    if cap:
        score = torch.tanh(score * (1.0 / cap)) * cap
    if slopes is not None:
        score = score - slopes * distance.abs().float()
    return score


def _weighted(score, seen):
    """Softmax over the last dimension of what is seen; zeros where nothing is."""
    score = torch.where(seen, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.where(seen, torch.exp(score - torch.where(top > float("-inf"), top, 0.0)), 0.0)
    total = weight.sum(-1, keepdim=True)
    return weight / torch.where(total > 0, total, 1.0)


def _sees(s, at, length, first, prefix, t):
    """Which tokens t a query sees; all of one shape but for the last dimension."""
    back = t <= at
    if s["case"]["window"]:
        back = back & (t > at - s["case"]["window"])
    seen = (t < length) & (back | (t < prefix) if prefix is not None else back)
    return seen & (t >= first) if first is not None else seen


def _gathered(s, pages):
    """[sequence, head, token, dim] in 32 bits of the pages that the tables name."""
    x = pages[s["table"].long()].float()
    b, w, h, ps, d = x.shape
    return x.transpose(1, 2).reshape(b, h, w * ps, d)


def _plain_prompt(s):
    c = s["case"]
    b, h, d = c["sequences"], c["heads"], c["dim"]
    g, m = c["q_heads"] // h, c["new"]
    dtype = s["q"].dtype
    # queries as rotated ones are held: rounded to their type
    q = _rotate(s, s["q"], s["at"]).to(dtype).float()
    wide = torch.zeros(b, m, h, g, d, device=q.device)
    wide[s["owner"], s["place"]] = q.view(-1, h, g, d)
    wide = wide.permute(0, 2, 3, 1, 4).reshape(b, h, g * m, d)

    def spread(x, fill=0):
        y = torch.full((b, m), fill, dtype=torch.int64, device=q.device)
        y[s["owner"], s["place"]] = x.long()
        return y[:, None, None, :, None]

    k, v = _gathered(s, s["k_pages"]), _gathered(s, s["v_pages"])
    n = k.shape[2]
    t = torch.arange(n, device=q.device)
    at = spread(s["at"], -1)
    seen = _sees(s, at, s["lengths"].view(b, 1, 1, 1, 1),
                 None if s["first"] is None else spread(s["first"]),
                 None if s["prefix"] is None else spread(s["prefix"]), t)
    score = torch.matmul(wide, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    slopes = None if s["slopes"] is None else s["slopes"].view(h, g, 1, 1)
    score = _shaped(s, score.view(b, h, g, m, n), at - t, slopes)
    out = torch.matmul(_weighted(score, seen).view(b, h, g * m, n), v)
    out = out.view(b, h, g, m, d).permute(0, 3, 1, 2, 4)
    return out[s["owner"], s["place"]].reshape(-1, h * g, d).to(dtype)


def _plain_token(s, k, v, length):
    """(outputs, weights [sequence, head, query head of it, token]); k, v [b, h, n, d]."""
    c = s["case"]
    b, h, d = c["sequences"], c["heads"], c["dim"]
    g, n = c["q_heads"] // h, k.shape[2]
    q = _rotate(s, s["q"], (length - 1).clamp(min=0)).reshape(b, h, g, d)
    t = torch.arange(n, device=q.device)
    at = (length.long() - 1).view(b, 1, 1, 1)
    first, prefix = (None if s.get(x) is None else s[x].view(b, 1, 1, 1)
                     for x in ("first", "prefix"))
    seen = _sees(s, at, length.view(b, 1, 1, 1), first, prefix, t)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    slopes = None if s["slopes"] is None else s["slopes"].view(h, g, 1)
    weight = _weighted(_shaped(s, score, at - t, slopes), seen)
    return torch.matmul(weight, v).reshape(b, h * g, d).to(s["q"].dtype), weight


def _to4(x):
    """Codes (two a byte, the first in the low bits) and scales of rows [..., dim]."""
    x = x.float()
    d = x.shape[-1]
    y = x.unflatten(-1, (d // BLOCK, BLOCK))
    top, e = torch.frexp(y.abs().amax(-1, keepdim=True))  # top in [0.5, 1)
    e = torch.where(top > 0.75, e - 2, e - 3)
    e = torch.where(top > 0, e, -125).clamp(-125, 125)
    a = torch.ldexp(y.abs(), -e)
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
            + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    code = (code + 8 * (y < 0).int()).flatten(-2)
    return ((code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8),
            (e[..., 0] + 127).to(torch.uint8))


def _from4(codes, scales):
    """The values of codes [..., dim / 2] and scales [..., dim / 32], in 32 bits."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    m = code & 7
    value = torch.where(m < 2, 0.5 * m, torch.ldexp(1.0 + 0.5 * (m & 1), (m >> 1) - 1))
    value = torch.where(code >= 8, -value, value).unflatten(-1, (-1, BLOCK))
    return torch.ldexp(value, scales[..., None].int() - 127).flatten(-2)


def _slots(s, owner, place):
    ps = s["case"]["page_size"]
    return s["table"][owner, place // ps].long(), place % ps


def _put4(s, k, v, owner, place):
    page, slot = _slots(s, owner, place)
    s["k_codes"][page, :, slot], s["k_scales"][page, :, slot] = _to4(k)
    s["v_codes"][page, :, slot], s["v_scales"][page, :, slot] = _to4(v)


def _held4(s):
    page, slot = _slots(s, s["owner"], s["place"])
    return (_from4(s["k_codes"][page, :, slot], s["k_scales"][page, :, slot]),
            _from4(s["v_codes"][page, :, slot], s["v_scales"][page, :, slot]))


def _gathered4(s):
    t = s["table"].long()
    b, w = t.shape
    h, ps, d = s["case"]["heads"], s["case"]["page_size"], s["case"]["dim"]
    k = _from4(s["k_codes"][t], s["k_scales"][t]).transpose(1, 2).reshape(b, h, w * ps, d)
    v = _from4(s["v_codes"][t], s["v_scales"][t]).transpose(1, 2).reshape(b, h, w * ps, d)
    return k, v


def _plain_evict(s):
    c = s["case"]
    keep, recent, ps = c["keep"], c["recent"], c["page_size"]
    weights = s["weights"].clone()
    b, h, capacity = weights.shape
    n = s["lengths"].long().view(b, 1, 1)
    t = torch.arange(capacity, device=weights.device)
    # the newest stand above every weight, tokens that are not there below
    rank = torch.where(t >= n - recent, float("inf"), weights.double())
    rank = torch.where(t < n, rank, float("-inf"))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(torch.arange(order.shape[-1], device=t.device) < n, order, capacity)
    kept = torch.full((b, h, keep), capacity, device=t.device)
    kept[..., :order.shape[-1]] = order.sort(-1).values
    there = kept < capacity
    over = n > keep  # the others stay as they are
    from_ = torch.where(there, kept, 0)
    moved = torch.where(there, weights.gather(2, from_), 0.0)
    compact = torch.zeros_like(weights)
    compact[..., :min(keep, capacity)] = moved[..., :capacity]
    weights = torch.where(over, compact, weights)
    # rows of kept tokens to the pages they move to
    seq = torch.arange(b, device=t.device).view(b, 1, 1).expand(b, h, keep)
    head = torch.arange(h, device=t.device).view(1, h, 1).expand(b, h, keep)
    page, slot = s["table"][seq, from_ // ps].long(), from_ % ps
    to = torch.arange(keep, device=t.device).expand(b, h, keep)
    to_page, to_slot = s["into"][seq, to // ps].long(), to % ps
    # a token that is not there writes back what its slot held
    page, slot = torch.where(there, page, to_page), torch.where(there, slot, to_slot)
    s["k_pages"][to_page, head, to_slot] = s["k_pages"][page, head, slot]
    s["v_pages"][to_page, head, to_slot] = s["v_pages"][page, head, slot]
    return torch.where(there, kept, -1).int(), weights, s["k_pages"], s["v_pages"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "prompt":
            return _plain_prompt(s)
        if kind == "evict":
            return _plain_evict(s)
        if kind in ("token", "weigh"):
            out, weight = _plain_token(s, _gathered(s, s["k_pages"]), _gathered(s, s["v_pages"]),
                                       s["lengths"])
            return out if kind == "token" else (out, s["weights"] + weight.sum(2))
        if kind == "append4":
            _put4(s, s["k"], s["v"], s["owner"], s["place"])
            return _held4(s)
        if kind == "attend4":
            return _plain_token(s, *_gathered4(s), s["lengths"])[0]
        _put4(s, s["k"], s["v"], s["owner"], s["place"])
        return (_plain_token(s, *_gathered4(s), s["lengths"] + 1)[0], *_held4(s))
    cache, table, lengths = s["cache"], s["table"], s["lengths"]
    if kind in ("prompt", "token", "weigh"):
        shape = dict(window=c["window"] or None, softcap=c["softcap"] or None, slopes=s["slopes"],
                     prefix=s["prefix"], first=s["first"])
        if kind == "prompt":
            return cache.attend(s["q"], table, lengths, s["offsets"], **shape)
        if kind == "token":
            return cache.attend(s["q"], table, lengths, **shape)
        weights = s["weights"].clone()
        return cache.attend(s["q"], table, lengths, weights=weights, **shape), weights
    if kind == "evict":
        weights = s["weights"].clone()
        kept = cache.evict(weights, table, lengths, c["keep"], recent=c["recent"],
                           into=s["into"])
        return kept, weights, s["k_pages"], s["v_pages"]
    if kind == "append4":
        cache.append(s["k"], s["v"], table, lengths, offsets=s["offsets"])
        return cache.read(s["k"].shape[0], table, lengths, offsets=s["offsets"])
    if kind == "attend4":
        return cache.attend(s["q"], table, lengths)
    out = cache.step(s["q"], s["k"], s["v"], table, lengths)
    return (out, *cache.read(c["sequences"], table, lengths))


# ---------------------------------------------------------------- in 64 bits

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _held_exact(x):
    """Rows as 4 bits hold them, in 64 bits: the nearest point of the grid times the least power
    of two that takes the block's largest to 6 or below; between two points, the even one."""
    d = x.shape[-1]
    y = x.double().reshape(-1, BLOCK)
    top = y.abs().amax(1, keepdim=True)
    power = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 6.0)))
    power = torch.where(top > 6 * power, 2 * power, power)  # log2 rounds
    power = torch.where(top <= 3 * power, power / 2, power)
    power = torch.where(top > 0, power, 1.0).clamp(2.0 ** -125, 2.0 ** 125)
    a = (y / power).abs()
    best, code = torch.zeros_like(a), torch.zeros_like(a)
    for i, point in enumerate(_GRID[1:], 1):
        off, was = (a - point).abs(), (a - best).abs()
        nearer = (off < was) | ((off == was) & (i % 2 == 0))
        best, code = torch.where(nearer, point, best), torch.where(nearer, float(i), code)
    return (torch.copysign(best, y) * power).reshape(*x.shape[:-1], d)


def _turned(c, x, at):
    """x [tokens, heads, dim] times exp(i angle); complex numbers do the rotation."""
    x = x.double()
    if not c["rotary"]:
        return x
    i = torch.arange(c["dim"] // 2, dtype=torch.float64)
    angle = at.cpu().double()[:, None] * torch.exp(-(2 * i / c["dim"]) * math.log(c["base"]))
    turn = torch.polar(torch.ones_like(angle), angle).cuda()[:, None]
    half = c["dim"] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * turn
    return torch.cat((z.real, z.imag), -1)


def _attended(c, q, k, v, at, first, prefix, slopes):
    """q [m, q_heads, dim] over k, v [h, n, dim], all in 64 bits: (out, weights summed over the
    queries and the query heads of a head [h, n]).  at, first, prefix [m]."""
    m, hq, d = q.shape
    h, n = k.shape[0], k.shape[1]
    g = hq // h
    out, mass = torch.zeros_like(q), torch.zeros(h, n, dtype=torch.float64, device=q.device)
    if n == 0:
        return out, mass
    t = torch.arange(n, device=q.device)[None]
    at, first, prefix = (x.to(q.device).long()[:, None] for x in (at, first, prefix))
    hidden = t > at
    if c["window"]:
        hidden = hidden | (t <= at - c["window"])
    hidden = (hidden & (t >= prefix)) | (t < first)
    nothing = hidden.all(1, keepdim=True)
    for j in range(hq):
        x = q[:, j] @ k[j // g].T.contiguous() / math.sqrt(d)
        if c["softcap"]:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        if slopes is not None:
            x = x - float(slopes[j]) * (at - t).abs().double()
        x = x.masked_fill(hidden, -math.inf)
        w = torch.softmax(x, 1).masked_fill(nothing, 0.0)
        out[:, j] = w @ v[j // g]
        mass[j // g] += w.sum(0)
    return out, mass


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    kind, ps = c["kind"], c["page_size"]
    lengths, new = _counts(c)
    if kind == "append4":
        return _held_exact(s["k"]), _held_exact(s["v"])
    if kind == "evict":
        kept = torch.full((len(lengths), c["heads"], c["keep"]), -1, dtype=torch.int32)
        weights, kp, vp = s["weights"].cpu().double(), s["k_pages"].double(), s["v_pages"].double()
        of = weights.tolist()
        for i, n in enumerate(lengths):
            old = max(0, n - c["recent"])
            for j in range(c["heads"]):
                w = of[i][j]
                # as many of the older tokens as the newest leave room for
                room = c["keep"] - (n - old)
                chosen = sorted(sorted(range(old), key=lambda t: (-w[t], t))[:room])
                chosen += range(old, n)
                kept[i, j, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
                if n > c["keep"]:
                    weights[i, j] = 0.0
                    weights[i, j, :len(chosen)] = torch.tensor([w[t] for t in chosen],
                                                               dtype=torch.float64)
                src, dst = torch.tensor(chosen, dtype=torch.int64), torch.arange(len(chosen))
                a, b = s["table"][i].cpu().long(), s["into"][i].cpu().long()
                for pages, held in ((kp, s["k_pages"]), (vp, s["v_pages"])):
                    rows = held[a[src // ps].cuda(), j, (src % ps).cuda()].double()
                    pages[b[dst // ps].cuda(), j, (dst % ps).cuda()] = rows
        return kept.cuda(), weights.cuda(), kp, vp
    four = kind in ("attend4", "step4")
    dtype = DTYPES[c["dtype"]]
    owner, at, _, first, prefix = _queries(c)
    if kind == "step4":
        at = at + 1
    q = _turned(c, s["q"], at.clamp(min=0))
    if kind == "prompt":
        q = q.to(dtype).double()
    outs, masses = [], []
    for i, n in enumerate(lengths):
        if four:
            a = int(s["old_offsets"][i])
            k, v = (_held_exact(s[x][a:a + n]) for x in ("old_k", "old_v"))
            if kind == "step4":
                k, v = (torch.cat((x, _held_exact(s[y][i:i + 1]))) for x, y in ((k, "k"), (v, "v")))
            k, v = k.transpose(0, 1), v.transpose(0, 1)
        else:
            n += new[i] if kind == "prompt" else 0
            used = s["table"][i, :(n + ps - 1) // ps].long()
            k, v = (s[x][used].double().transpose(0, 1).flatten(1, 2)[:, :n]
                    for x in ("k_pages", "v_pages"))
        of = (owner == i) if kind == "prompt" else torch.arange(len(lengths)) == i
        out, mass = _attended(c, q[of.cuda()], k, v, at[of], first[of], prefix[of], s["slopes"])
        outs.append(out)
        masses.append(mass)
    out = torch.cat(outs)
    if kind == "step4":
        return out, _held_exact(s["k"]), _held_exact(s["v"])
    if kind != "weigh":
        return out
    weights = s["weights"].double()
    for i, mass in enumerate(masses):
        weights[i, :, :mass.shape[1]] += mass
    return out, weights
