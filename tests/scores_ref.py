"""Attention over pages with scores of its own in 64 bits, on the CPU, with the tolerances that
the arithmetic allows (derived here, before any run), and a helper that keeps sequences in pages.

u(T) = finfo(T).eps / 2 is the relative error of one rounding to T.
"""
import math
import random

import torch

import paged_ref as R

U32 = 2.0 ** -24


def sees(n, at, first, prefix, window):
    """[m, n]: which tokens each query sees."""
    t = torch.arange(n)[None]
    at, first, prefix = (x.long()[:, None] for x in (at, first, prefix))
    back = t <= at
    if window:
        back &= t > at - window
    return (t >= first) & (back | (t < prefix))


def rounded(x, err, dtype):
    """x (fp64, computed with up to `err`) rounded to a type: (values, how far a computed one may
    round elsewhere)."""
    lo, hi = (x - err).to(dtype).double(), (x + err).to(dtype).double()
    return x.to(dtype).double(), (hi - lo).abs()


def attend(q, k, v, seen, at, scale, dtype, *, softcap=None, slopes=None, q_err=None, rough=False):
    """q [m, Hq, D] fp64 over k, v [H, n, D]: (out [m, Hq, D], tolerance, weights [H, n] summed over
    queries and query heads, tolerance).

    A score is off by d: 2^-24 scale sum|q k| (8 + 4 sqrt(D)) (rounding errors of a sum of D
    terms add as a random walk; 4 standard deviations), 16 * 2^-24 of itself and of its bias for
    the exponent's argument, the bias' factor and its product, scale sum|k| q_err for the query's
    own error; the cap's slope is at most 1 and tanh itself is off by 2^-21 of its value (rough,
    half-precision prompts: by 2^-21 of the cap).  That is a relative error of 2 d in a weight
    over its sum.  Exponential, product, quotient and joins round a few times each (32), the sum
    over n tokens as a random walk (4 sqrt(n)).  Weights and queries enter half-precision products
    as two numbers at the least: 2^-16 of the value (bf16), 2^-20 (fp16).  Then the rounding to
    the type.

    A weight exp(s - m) below 2^-126, fp32's smallest normal number, is 0, and so is what a
    number of a weight, or a product of one and a value, has below it: with up to three numbers a
    weight, that is up to 2^-126 (1 + 3 |v|) of each token's part, over a sum of 1 or more.  It
    shows where everything else of an output is 0: one token of value 0 beside others of weight
    1e-40 gave 0 for -2e-40."""
    m, hq, d = q.shape
    h, n = k.shape[:2]
    g = hq // h
    k, v = k.double(), v.double()
    out, tol = torch.zeros(m, hq, d, dtype=torch.float64), torch.zeros(m, hq, d, dtype=torch.float64)
    mass, mass_tol = (torch.zeros(h, n, dtype=torch.float64) for _ in range(2))
    if n == 0 or m == 0:
        return out, tol, mass, mass_tol
    split = {torch.float32: 0.0, torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -16}[dtype]
    none = ~seen.any(1, keepdim=True)
    t = torch.arange(n)[None]
    for j in range(hq):
        kj, vj = k[j // g], v[j // g]
        s = q[:, j] @ kj.T * scale
        size = q[:, j].abs() @ kj.abs().T * abs(scale)
        ds = size * (U32 * (8 + 4 * math.sqrt(d)) + split)
        if q_err is not None:
            ds = ds + q_err[:, j] @ kj.abs().T * abs(scale)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
            ds = ds + 2.0 ** -21 * (softcap if rough else s.abs())
        bias = torch.zeros_like(s)
        if slopes is not None:
            bias = float(slopes[j]) * (at[:, None] - t).abs().double()
        s = s - bias
        ds = ds + 16 * U32 * (s.abs() + bias)
        w = torch.softmax(s.masked_fill(~seen, -math.inf), 1).masked_fill(none, 0.0)
        # tokens of no weight to speak of do not count for the largest error
        ds = (ds * (w > 1e-12)).amax(1, keepdim=True)
        rel = 2 * ds + U32 * (32 + 4 * math.sqrt(n)) + split
        out[:, j] = w @ vj
        lost = 2.0 ** -126 * (seen.double() @ (1 + 3 * vj.abs()))
        tol[:, j] = rel * (w @ vj.abs()) + lost + R.u(dtype) * out[:, j].abs() + R._tiny(dtype)
        mass[j // g] += w.sum(0)
        mass_tol[j // g] += (w * rel).sum(0) + 1e-12
    return out, tol, mass, mass_tol


class Pool:
    """Sequences in pages: tables, lengths, and the rows as the 64-bit side sees them."""

    def __init__(self, lengths, heads, dim, page_size, dtype, *, seed=0, spare=3, extra=0,
                 fill=float("nan"), rows=True):
        self.g = torch.Generator().manual_seed(seed)
        self.heads, self.dim, self.ps, self.dtype = heads, dim, page_size, dtype
        need = [-(-(n + extra) // page_size) for n in lengths]
        self.pages = sum(need) + spare
        order = list(range(self.pages))
        random.Random(seed).shuffle(order)
        width = max(1, max(need))
        # entries behind a sequence's pages hold anything
        self.table_host = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(lengths), width + 2),
                                        generator=self.g, dtype=torch.int64).int()
        at = 0
        for i, n in enumerate(need):
            self.table_host[i, :n] = torch.tensor(order[at:at + n])
            at += n
        self.free = order[at:]
        self.table = self.table_host.cuda()[:, :width]
        self.held = list(lengths)
        self.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
        if rows:
            shape = (self.pages, heads, page_size, dim)
            self.k_pages, self.v_pages = (torch.full(shape, fill, dtype=dtype, device="cuda")
                                          for _ in range(2))
            self.k = [self.normal(n, heads, dim) for n in lengths]
            self.v = [self.normal(n, heads, dim) for n in lengths]
            for i in range(len(lengths)):
                self.put(i)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dtype)

    def put(self, i):
        p = torch.arange(self.k[i].shape[0])
        page, slot = self.table_host[i, p // self.ps].long().cuda(), (p % self.ps).cuda()
        self.k_pages[page, :, slot] = self.k[i].cuda()
        self.v_pages[page, :, slot] = self.v[i].cuda()


def spans(counts):
    """int32 offsets of so many tokens each, on the GPU."""
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32).cuda()
