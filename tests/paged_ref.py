"""Rotary positions and attention over pages in 64 bits, on the CPU, with the
tolerances that the arithmetic allows (derived here, before any run).

u(T) = finfo(T).eps / 2 is the relative error of one rounding to T.
"""
import math

import torch

U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def frequencies(dim, base=10000.0, scaling=None, factor=1.0, context=0, slow=None, fast=None,
                amplitude=None):
    """(angles per position [dim/2] fp64, amplitude)."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (dim / (dim - 2))
    f = torch.tensor(base, dtype=torch.float64) ** (-2 * i / dim)
    slow = slow or 1.0
    fast = fast or (32.0 if scaling == "yarn" else 4.0)
    amp = 1.0
    keep = torch.ones_like(f)
    if scaling == "linear":
        keep = torch.zeros_like(f)
    elif scaling == "bands":
        keep = ((context * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
    elif scaling == "yarn":
        pair = [dim * math.log(context / (n * 2 * math.pi)) / (2 * math.log(base))
                for n in (fast, slow)]
        lo, hi = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), dim - 1)
        keep = (1 - (i - lo) / (hi - lo if hi > lo else 0.001)).clamp(0, 1)
        amp = 0.1 * math.log(factor) + 1
    return keep * f + (1 - keep) * f / factor, amp if amplitude is None else amplitude


def rotate(x, positions, dim, interleaved=False, backward=False, **kw):
    """x [..., heads, D] at positions [...]: (rotated fp64, error allowed).

    Each member is x1 c - x2 s.  Cosine and sine come with up to 2 ulp of 1 (2^-23) from
    the function and 0.8 * 2^-24 from its argument's rounding (an angle of at most pi / 4);
    the amplitude and its product, the member's product and the sum round once each:
    (4 + 0.8 + 1 + 1 + 1 + 1) 2^-24 < 2^-20 of a (|x1| + |x2|), then the rounding to the
    type.  The angle's 2^-33 of a turn is a thousandth of that."""
    f, amp = frequencies(dim, **kw)
    x64 = x.detach().cpu().double()
    angle = positions.cpu().double()[..., None] * f
    c, s = (t(angle)[..., None, :] * amp for t in (torch.cos, torch.sin))
    if backward:
        s = -s
    p = dim // 2
    if interleaved:
        a, b = x64[..., 0:dim:2], x64[..., 1:dim:2]
    else:
        a, b = x64[..., :p], x64[..., p:dim]
    y1, y2, size = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * amp
    y, e = x64.clone(), torch.zeros_like(x64)
    if interleaved:
        y[..., 0:dim:2], y[..., 1:dim:2] = y1, y2
        e[..., 0:dim:2] = e[..., 1:dim:2] = size
    else:
        y[..., :p], y[..., p:dim] = y1, y2
        e[..., :p] = e[..., p:dim] = size
    tol = e * 2.0 ** -20
    tol[..., :dim] += u(x.dtype) * y[..., :dim].abs() + _tiny(x.dtype)
    return y, tol


def _tiny(dtype):
    """Half the spacing of the smallest numbers of a type."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def attend(q, k, v, scale, dtype, q_err=0.0):
    """One query a head over all of k, v: q [H, g, D] fp64, k, v [H, n, D]: (out fp64 [H, g,
    D], error allowed).

    The weights are exp(s_t - max) / sum.  A score is off by d = 2^-24 scale sum|q k| (8 +
    4 sqrt(D)) (rounding errors of a sum of D terms add as a random walk; 4 standard
    deviations) plus 2^-24 |s| (16) for the exponent's argument, plus scale * q_err sum|k| for
    the rotated query's own error; that is a relative error of 2 d in a weight over its sum.
    The exponential, the product with v, the quotient and the joins of the parts round a few
    times each (32), the sum over n tokens as a random walk (4 sqrt(n)).  Weights and queries
    enter the matrix cores as two half-precision numbers, the largest below and the rest: the
    rest is up to 2^-7 of it (bf16) and rounds by 2^-9 of that, 2^-16 of the value; fp16 2^-10
    and 2^-10, 2^-20 (the rounding of a rest below its normal numbers is 2^-40 of the largest
    weight, nothing).  Then the rounding to the type."""
    q, k, v = q.double(), k.double(), v.double()
    n, d = k.shape[1], k.shape[2]
    if n == 0:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, z
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    w = torch.softmax(s, -1)
    out = torch.matmul(w, v)
    size = torch.matmul(q.abs(), k.abs().transpose(1, 2)) * abs(scale)
    split = {torch.float32: 0.0, torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -16}[dtype]
    ds = size * (U32 * (8 + 4 * math.sqrt(d)) + split) + 16 * U32 * s.abs()
    if not isinstance(q_err, float):
        ds = ds + torch.matmul(q_err, k.abs().transpose(1, 2)) * abs(scale)
    ds = ds.amax(-1, keepdim=True)
    rel = 2 * ds + U32 * (32 + 4 * math.sqrt(n)) + split
    return out, rel * torch.matmul(w, v.abs()) + u(dtype) * out.abs() + _tiny(dtype)


def check(got, want, tol, what=""):
    got = got.detach().cpu().double()
    err = (got - want).abs()
    bad = ~(err <= tol)  # also where got is NaN
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: "
                             f"{got[i].item()!r} for {want[i].item()!r}, allowed {tol[i].item():.3g}")
