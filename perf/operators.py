"""Rotary positions, the paged cache and its single-token attention: cases and plain forms.

A case is one call of one operator on one shape:

  rotary   queries and keys rotated by their tokens' positions, with the gradient if asked for
  append   keys (rotated on the way) and values written into the pages of their sequences
  attend   one new token per sequence attends over its sequence's pages
  step     a decode step: one token per sequence appended, then its attention

``listed`` holds the sizes of the repository's own configurations and what lies
between them, ``draw`` more of the same ranges.  ``run`` computes the operators
in elementary torch operations where ``own`` is false, and through the library
where it is true; ``exact`` restates them in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(kind, **kw):
    c = dict(kind=kind, sequences=1, tokens=1, least=0, new=1, q_heads=8, heads=8, dim=128,
             page_size=16, dtype="bfloat16", rotary_dim=0, interleaved=False, base=10000.0,
             scaling="", factor=1.0, context=0, first=0, window=0, gradient=False)
    c.update(kw)
    return c


def listed():
    return [
        # a chat's next token on a 24-layer stack of 14 heads: latency alone
        _case("rotary", name="rotary_token", q_heads=14, heads=14, dim=64, rotary_dim=64,
              dtype="float16", first=511),
        # a prompt of a model with grouped heads whose context was stretched by wavelength bands
        _case("rotary", name="rotary_prompt", tokens=8192, q_heads=32, heads=8, rotary_dim=128,
              base=500000.0, scaling="bands", factor=8.0, context=8192),
        # a training step's forward and backward: a batch of odd length whose queries and keys
        # are views of one projection, interleaved pairs on half of each head, far positions
        _case("rotary", name="rotary_train", sequences=3, tokens=1277, q_heads=16, heads=4,
              dim=128, rotary_dim=64, interleaved=True, dtype="float32", scaling="yarn",
              factor=16.0, context=8192, first=120000, gradient=True),
        # one token of each of 64 running sequences
        _case("append", name="append_token", sequences=64, tokens=1280, least=16,
              rotary_dim=128),
        # ragged prompts arriving together, some behind a cached beginning; fp32 rows, part of each
        # head rotated
        _case("append", name="append_prompts", sequences=16, tokens=640, least=0, new=2048,
              heads=4, dim=80, page_size=32, dtype="float32", rotary_dim=32, interleaved=True),
        # one long prompt
        _case("append", name="append_long", tokens=0, new=40000, page_size=64, rotary_dim=128),
        # a server's ragged batch, an empty sequence in it, 8 query heads per key head
        _case("attend", name="attend_ragged", sequences=16, tokens=1280, least=0, q_heads=32,
              heads=4, dim=64, dtype="float16", rotary_dim=64),
        # one long sequence: few rows, split over its length
        _case("attend", name="attend_long", tokens=32768, least=32768, q_heads=32, rotary_dim=128,
              page_size=64),
        # fp32 rows, a head dimension that is no power of two, a sliding window, odd lengths
        _case("attend", name="attend_window", sequences=7, tokens=4001, least=33, q_heads=12,
              heads=4, dim=96, page_size=48, dtype="float32", window=1000),
        # one layer of 64 sequences of 8,192 tokens: the memory's rate
        _case("attend", name="attend_batch", sequences=64, tokens=8192, least=8192, q_heads=32,
              rotary_dim=128, page_size=64),
        # a chat's decode step as one call
        _case("step", name="step_token", tokens=511, q_heads=14, heads=2, dim=64,
              dtype="float16", rotary_dim=64),
        # a decode step of a server's ragged batch
        _case("step", name="step_ragged", sequences=32, tokens=2048, least=0, q_heads=32,
              rotary_dim=128, page_size=32, base=500000.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "append", "append", "attend", "attend", "attend",
                       "step", "step"))
    heads = rng.choice((1, 2, 4, 4, 8, 8, 14))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 256))
    c = dict(heads=heads, dim=dim, dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
             q_heads=heads * rng.choice((1, 2, 3, 4, 4, 7, 8)),
             page_size=rng.choice((16, 16, 32, 48, 64, 128, 256)),
             rotary_dim=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.3,
             base=rng.choice((10000.0, 500000.0, 1000000.0)))
    c["scaling"] = rng.choice(("", "", "linear", "ntk", "yarn", "bands"))
    if c["scaling"]:
        c.update(factor=rng.choice((2.0, 4.0, 8.0, 32.0)), context=rng.choice((2048, 4096, 8192)))
    if kind == "rotary":
        tokens, sequences = _spread(rng, 1, 8192), _spread(rng, 1, 8)
        while sequences * tokens * (c["q_heads"] + heads) * dim > 1 << 25:
            tokens = max(1, tokens // 2)
        return _case(kind, **{**c, "sequences": sequences, "tokens": tokens,
                              "first": rng.choice((0, 0, _spread(rng, 1, 1000000))),
                              "gradient": rng.random() < 0.4})
    if kind == "append":
        tokens, new = _spread(rng, 1, 4096), rng.choice((1, _spread(rng, 2, 40000)))
        sequences = _spread(rng, 1, 256)
        while sequences > 1 and sequences * (tokens + new) * heads * dim > 1 << 26:
            sequences //= 2
        return _case(kind, **{**c, "sequences": sequences, "tokens": tokens, "new": new,
                              "least": rng.choice((0, tokens))})
    tokens = _spread(rng, 1, 65536)
    sequences = _spread(rng, 1, 128)
    while sequences * tokens * heads * dim > (1 << 28 if kind == "attend" else 1 << 25):
        sequences, tokens = max(1, sequences // 2), max(1, tokens * 3 // 4)
    return _case(kind, **{**c, "sequences": sequences, "tokens": tokens,
                          "least": rng.choice((0, 1, tokens // 4, tokens)),
                          "window": rng.choice((0, 0, 0, _spread(rng, 1, 4096)))})


# ---------------------------------------------------------------- the shapes

def _counts(c):
    """Per sequence: the tokens it holds before the call, and the new ones."""
    rng = random.Random(c["tokens"] * 1000003 + c["sequences"])
    lengths = [rng.randint(c["least"], c["tokens"]) for _ in range(c["sequences"])]
    lengths[0], lengths[-1] = c["least"], c["tokens"]
    new = [rng.randint(1, c["new"]) for _ in lengths]
    new[0] = c["new"]
    return lengths, new


def work(c):
    size = 4 if c["dtype"] == "float32" else 2
    row = c["dim"] * size
    if c["kind"] == "rotary":
        n = c["sequences"] * c["tokens"] * (c["q_heads"] + c["heads"])
        passes = 2 if c["gradient"] else 1
        return {"bytes": passes * (2 * n * row + 4 * c["tokens"]),
                "flops": passes * 3 * n * c["rotary_dim"]}
    lengths, new = _counts(c)
    b, total = c["sequences"], sum(new)
    write = 4 * total * c["heads"] * row
    turn = 3 * c["rotary_dim"]
    if c["kind"] == "append":
        return {"bytes": write + 8 * b, "flops": turn * total * c["heads"]}
    step = c["kind"] == "step"
    seen = [n + 1 if step else n for n in lengths]
    seen = sum(min(n, c["window"]) if c["window"] else n for n in seen)
    # the step's own token is read from its input: its row is written, not read back
    rows = 2 * (seen - b if step else seen) * c["heads"]
    io = 2 * b * c["q_heads"] * row
    return {"bytes": rows * row + io + (write if step else 0) + 8 * b,
            "flops": 4 * seen * c["q_heads"] * c["dim"] + turn * b * c["q_heads"]
            + (turn * b * c["heads"] if step else 0)}


# ---------------------------------------------------------------- the inputs

def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    rng = random.Random(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    if c["kind"] == "rotary":
        b, t, hq, hk = c["sequences"], c["tokens"], c["q_heads"], c["heads"]
        first = c["first"] + rng.randint(0, 15)
        s = {"positions": torch.arange(first, first + t, device="cuda", dtype=torch.int32)}
        qkv = normal(b, t, hq + 2 * hk, c["dim"])  # one projection's output
        s["q"], s["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
        if c["gradient"]:
            s["q"].requires_grad_()
            s["k"].requires_grad_()
            s["dq"], s["dk"] = normal(b, t, hq, c["dim"]), normal(b, t, hk, c["dim"])
        return s
    lengths, new = _counts(c)
    ps = c["page_size"]
    extra = [0 if c["kind"] == "attend" else n for n in new]
    need = [(n + e + ps - 1) // ps for n, e in zip(lengths, extra)]
    # the pool of a server: some pages are free, a sequence's lie anywhere
    pages = sum(need) + 8
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.zeros(c["sequences"], max(1, max(need)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s = {"table": table.cuda(), "held": lengths, "new": new,
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    # heads differ in scale, as the keys and values of a model do
    scale = torch.exp(0.5 * torch.randn(2, c["heads"], 1, 1, generator=g, device="cuda")).to(dtype)
    s["k_pages"] = normal(pages, c["heads"], ps, c["dim"]).mul_(scale[0])
    s["v_pages"] = normal(pages, c["heads"], ps, c["dim"]).mul_(scale[1])
    if c["kind"] != "append":
        s["q"] = normal(c["sequences"], c["q_heads"], c["dim"])
    if c["kind"] != "attend":
        total = sum(new)
        s["k"] = normal(total, c["heads"], c["dim"]).mul_(scale[0, :, :, 0])
        s["v"] = normal(total, c["heads"], c["dim"]).mul_(scale[1, :, :, 0])
        if c["new"] > 1:  # where each sequence's new tokens begin
            s["offsets"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)],
                                        dtype=torch.int32, device="cuda")
        # what a program that places the tokens itself keeps beside them
        s["owner"] = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], device="cuda")
        s["place"] = torch.tensor([lengths[i] + j for i, n in enumerate(new) for j in range(n)],
                                  device="cuda")
    return s


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if own:
        from adaptq_amd.paged import PagedCache
        from adaptq_amd.rotary import Rotary
        rotary = None
        if c["rotary_dim"]:
            rotary = Rotary(c["rotary_dim"], base=c["base"], interleaved=c["interleaved"],
                            scaling=c["scaling"] or None, factor=c["factor"],
                            context=c["context"])
        s["rotary"] = rotary
        if c["kind"] != "rotary":
            s["cache"] = PagedCache(s["k_pages"], s["v_pages"], rotary=rotary)
    elif c["rotary_dim"]:
        f, a = _frequencies(c)
        s["frequencies"], s["amplitude"] = torch.tensor(f, dtype=torch.float64, device="cuda"), a
    return s


# ---------------------------------------------------------------- the plain forms

def _frequencies(c):
    """Angle per position of each pair, and the factor on cosine and sine."""
    r, base, s = c["rotary_dim"], c["base"], c["factor"]
    f = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if c["scaling"] == "linear":
        return [x / s for x in f], 1.0
    if c["scaling"] == "ntk":
        wide = base * s ** (r / (r - 2.0))
        return [wide ** (-2.0 * i / r) for i in range(r // 2)], 1.0
    if c["scaling"] == "bands":
        # pairs that turn over 4 times in the context stay, those below once slow down
        keep = [(c["context"] * x / (2 * math.pi) - 1.0) / 3.0 for x in f]
    elif c["scaling"] == "yarn":
        # a ramp over the pairs between the ones that turn 32 times and once in the context
        low, high = (r * math.log(c["context"] / (n * 2 * math.pi)) / (2 * math.log(base))
                     for n in (32, 1))
        low, high = max(0, math.floor(low)), min(r - 1, math.ceil(high))
        keep = [1.0 - (i - low) / (high - low if high > low else 0.001) for i in range(r // 2)]
    else:
        return f, 1.0
    keep = [min(1.0, max(0.0, t)) for t in keep]
    amplitude = 0.1 * math.log(s) + 1.0 if c["scaling"] == "yarn" and s > 1 else 1.0
    return [x * (t + (1 - t) / s) for x, t in zip(f, keep)], amplitude


def _rotate(s, x, positions):
    """x [..., heads, dim] at positions [...], in 32 bits."""
    c = s["case"]
    x = x.float()
    if not c["rotary_dim"]:
        return x
    angle = positions.double()[..., None] * s["frequencies"]
    cos = (torch.cos(angle) * s["amplitude"]).float()[..., None, :]
    sin = (torch.sin(angle) * s["amplitude"]).float()[..., None, :]
    r = c["rotary_dim"]
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1) if r < c["dim"] else turned


def _plain_rotary(s):
    dtype = s["q"].dtype
    q = _rotate(s, s["q"], s["positions"]).to(dtype)
    k = _rotate(s, s["k"], s["positions"]).to(dtype)
    if not s["case"]["gradient"]:
        return q, k
    return (q.detach(), k.detach(),
            *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))


def _plain_append(s):
    ps = s["case"]["page_size"]
    page = s["table"][s["owner"], s["place"] // ps].long()
    slot = s["place"] % ps
    s["k_pages"][page, :, slot] = _rotate(s, s["k"], s["place"]).to(s["k_pages"].dtype)
    s["v_pages"][page, :, slot] = s["v"]


def _plain_attend(s, seen):
    """One query a sequence over its first `seen` tokens."""
    c = s["case"]
    b, h, d, ps = c["sequences"], c["heads"], c["dim"], c["page_size"]
    g, width = c["q_heads"] // h, s["table"].shape[1]
    q = _rotate(s, s["q"], seen - 1).reshape(b, h, g, d)
    table = s["table"].long()
    # [sequence, page, head, slot, dim] -> [sequence, head, token, dim]
    k = s["k_pages"][table].float().transpose(1, 2).reshape(b, h, width * ps, d)
    v = s["v_pages"][table].float().transpose(1, 2).reshape(b, h, width * ps, d)
    score = torch.matmul(k, q.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    at = torch.arange(width * ps, device=q.device)
    inside = at < seen[:, None]
    if c["window"]:
        inside &= at >= seen[:, None] - c["window"]
    inside = inside[:, None, :, None]
    score = torch.where(inside, score, float("-inf"))
    top = score.amax(2, keepdim=True)
    weight = torch.where(inside, torch.exp(score - top), 0.0)
    total = weight.sum(2)
    out = torch.matmul(weight.transpose(2, 3).contiguous(), v) / total[..., None]
    out = torch.where((seen > 0)[:, None, None, None], out, 0.0)
    return out.reshape(b, h * g, d).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["kind"] == "rotary":
            return _plain_rotary(s)
        if c["kind"] == "attend":
            return _plain_attend(s, s["lengths"])
        _plain_append(s)
        if c["kind"] == "append":
            return s["k_pages"], s["v_pages"]
        return _plain_attend(s, s["lengths"] + 1), s["k_pages"], s["v_pages"]
    if c["kind"] == "rotary":
        q, k = s["rotary"](s["positions"], s["q"], s["k"])
        if not c["gradient"]:
            return q, k
        return (q.detach(), k.detach(),
                *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    cache, window = s.get("cache"), c["window"] or None
    if c["kind"] == "append":
        cache.append(s["k"], s["v"], s["table"], s["lengths"], offsets=s.get("offsets"))
        return s["k_pages"], s["v_pages"]
    if c["kind"] == "attend":
        return cache.attend(s["q"], s["table"], s["lengths"], window=window)
    out = cache.step(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=window)
    return out, s["k_pages"], s["v_pages"]


# ---------------------------------------------------------------- in 64 bits

def _turns(c, positions):
    """exp(i angle) of every position and pair, in 64 bits, times the amplitude."""
    r = c["rotary_dim"]
    i = torch.arange(r // 2, dtype=torch.float64)
    base = c["base"] * (c["factor"] ** (r / (r - 2)) if c["scaling"] == "ntk" else 1.0)
    f = torch.exp(-(2 * i / r) * math.log(base))
    amplitude = 1.0
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] in ("bands", "yarn"):
        over = c["context"] * f / (2 * math.pi)  # turns over the original context
        if c["scaling"] == "bands":
            keep = ((over - 1) / (4 - 1)).clamp(0, 1)
        else:
            # the pair (a real number) that turns n times over the context
            lo, hi = ((math.log(c["context"] / (2 * math.pi)) - math.log(n)) * r
                      / (2 * math.log(c["base"])) for n in (32, 1))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
            keep = 1 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            amplitude += 0.1 * math.log(max(c["factor"], 1.0))
        f = keep * f + (1 - keep) * f / c["factor"]
    angle = positions.cpu().double()[:, None] * f
    return torch.polar(torch.full_like(angle, amplitude), angle).cuda()


def _turned(c, x, turns):
    """x [tokens, heads, dim] times turns [tokens, pairs]; complex numbers do the rotation."""
    x, r = x.double(), c["rotary_dim"]
    if not r:
        return x
    z = x[..., :r]
    z = torch.complex(*(z.unflatten(-1, (r // 2, 2)).unbind(-1) if c["interleaved"]
                        else z.unflatten(-1, (2, r // 2)).unbind(-2))) * turns[:, None]
    z = torch.stack((z.real, z.imag), -1 if c["interleaved"] else -2).flatten(-2)
    return torch.cat((z, x[..., r:]), -1)


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    with torch.no_grad():
        if c["kind"] == "rotary":
            turns = _turns(c, s["positions"])
            names = ("q", "k", "dq", "dk") if c["gradient"] else ("q", "k")
            return tuple(torch.stack([_turned(c, x, turns.conj() if n[0] == "d" else turns)
                                      for x in s[n]]) for n in names)
        ps, rot = c["page_size"], c["rotary_dim"]
        kp, vp = s["k_pages"], s["v_pages"]
        at = 0
        if c["kind"] != "attend":
            kp, vp = kp.double(), vp.double()
            for i, (n, m) in enumerate(zip(s["held"], s["new"])):
                p = torch.arange(n, n + m)
                k = _turned(c, s["k"][at:at + m], _turns(c, p) if rot else None)
                page, slot = s["table"][i].cpu().long()[p // ps].cuda(), (p % ps).cuda()
                kp[page, :, slot] = k
                vp[page, :, slot] = s["v"][at:at + m].double()
                at += m
            if c["kind"] == "append":
                return kp, vp
        # the attention reads the rows as the pages hold them, rounded to their type
        dtype = DTYPES[c["dtype"]]
        outs = []
        for i, n in enumerate(s["held"]):
            n += c["kind"] == "step"
            if n == 0:
                outs.append(torch.zeros(c["q_heads"], c["dim"], dtype=torch.float64,
                                        device="cuda"))
                continue
            used = s["table"][i, :(n + ps - 1) // ps].long()
            lo = max(0, n - c["window"]) if c["window"] else 0
            k, v = (x[used].to(dtype).double().transpose(0, 1).flatten(1, 2)[:, lo:n]
                    for x in (kp, vp))
            q = _turned(c, s["q"][i:i + 1], _turns(c, torch.tensor([n - 1])) if rot else None)[0]
            q = q.view(c["heads"], -1, c["dim"])
            w = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(c["dim"]), -1)
            outs.append(torch.einsum("hgn,hnd->hgd", w, v).flatten(0, 1))
        out = torch.stack(outs)
        return out if c["kind"] == "attend" else (out, kp, vp)
