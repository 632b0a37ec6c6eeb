"""What the paged attention holds its queries and weights to: rotated fp16 queries of any size,
and bf16 queries and weights in fp32, against the formula in 64 bits with bounds derived here."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
U = R.U32


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    globals().update(PagedCache=PagedCache, Rotary=Rotary)


def _cache(k, v, rotary=None, page=16):
    """A cache that holds one sequence, k and v [tokens, heads, dim] as its pages have them."""
    n, heads, dim = k.shape
    pages = (n + page - 1) // page
    pools = []
    for x in (k, v):
        p = torch.zeros(pages * page, heads, dim, dtype=k.dtype)
        p[:n] = x
        pools.append(p.view(pages, page, heads, dim).transpose(1, 2).contiguous().cuda())
    table = torch.arange(pages, dtype=torch.int32).cuda()[None]
    return (PagedCache(*pools, rotary=rotary), table,
            torch.tensor([n], dtype=torch.int32).cuda())


def _check(q, k, v, rot=0, scale=None, **kw):
    """attend of q [1, q_heads, dim] against the formula, with the bounds of paged_ref."""
    n, heads, dim = k.shape
    cache, table, lengths = _cache(k, v, Rotary(rot, **kw) if rot else None)
    got = cache.attend(q.cuda(), table, lengths, scale=scale)
    x, err = q.double(), 0.0
    if rot:
        x, err = R.rotate(q.float(), torch.tensor([n - 1]), rot, **kw)
        err = err[0].view(heads, -1, dim)
    o, t = R.attend(x[0].view(heads, -1, dim), k.transpose(0, 1), v.transpose(0, 1),
                    scale if scale is not None else 1 / math.sqrt(dim), k.dtype, err)
    R.check(got[0], o.reshape(-1, dim), t.reshape(-1, dim))


@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -8, 2.0 ** -12, 2.0 ** -15])
def test_small_fp16_queries(size, dim):
    """Queries of 2^-8 to 2^-15 against keys that are as much larger: a query's two halves keep
    2^-20 of its row's largest value, not 2^-24 of 1."""
    g = torch.Generator().manual_seed(dim)
    normal = lambda *shape: torch.randn(shape, generator=g)  # noqa: E731
    k = (normal(64, 2, dim) / size * 0.25).half()
    v = normal(64, 2, dim).half()
    q = (normal(1, 12, dim) * size * 4).half()
    _check(q, k, v, rot=dim // 2, base=100.0)


@pytest.mark.parametrize("amplitude", [0.001, 4.0, 1e10, 1e30])
@pytest.mark.parametrize("dim", [64, 128])
def test_amplitudes_take_fp16_queries_anywhere(amplitude, dim):
    """A rotated query beyond 131,008 (the most that two fp16 numbers add up to), or far below
    fp16's normal numbers, scores as the formula says."""
    g = torch.Generator().manual_seed(dim)
    normal = lambda *shape: torch.randn(shape, generator=g)  # noqa: E731
    k, v = normal(80, 1, dim).half(), normal(80, 1, dim).half()
    q = (normal(1, 5, dim) * 15000).clamp(-60000, 60000).half()
    _check(q, k, v, rot=dim, amplitude=amplitude, scale=1 / (15000 * math.sqrt(dim) * amplitude))


def test_one_large_channel():
    """Rows of one query that differ by 2^20: each is scaled by its own largest value, and the
    small channels of a row keep their share of its score."""
    g = torch.Generator().manual_seed(1)
    normal = lambda *shape: torch.randn(shape, generator=g)  # noqa: E731
    k, v = normal(40, 1, 64).half(), normal(40, 1, 64).half()
    q = normal(1, 16, 64)
    q *= 2.0 ** torch.linspace(-12, 10, 16)[None, :, None]
    q[0, 3::4, 5] *= 30
    k[:, :, 5] = (k[:, :, 5].float() / 30).half()
    _check(q.half(), k, v, rot=32, amplitude=1.5, scale=0.01)


def _cancelled(w, v):
    """v [n, dim] with its last four rows such that sum w v is 0 but for a rounding of a rounding
    of a rounding of bf16: what the output's own rounding hides is in plain sight."""
    v = v.clone()
    v[-4:] = 0
    for t in range(-1, -5, -1):
        v[t] = (-(w @ v.double()) / w[t]).to(v.dtype)
    return v


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("seed", range(4))
def test_bf16_weights(dim, seed):
    """Weights of bf16 pages hold fp32's 24 bits.  A score here is one product, q_0 k_0 (bf16 x
    bf16: exact) times scale (a power of two) and log2(e): with |s| <= 1 off by 2^-23 |s| for the
    constant and its product; less the largest, 2^-24 of up to 2; all of it into the weight as
    ln 2 at most, (2 + 2) 2^-24 and as much for the largest's own, and the exponential by 2^-23:
    10 * 2^-24.  The sums over 20 tokens (two units' halves) and the quotient round some 20 times
    by at most 2^-24 of sum |w v|, the weights' three parts leave 2^-24: 31 in all, so 2^-19
    covers them; the sum of the weights, off as much, scales an output near 0.  A weight held to
    2^-16 would be off by up to 8 times that."""
    g = torch.Generator().manual_seed(seed)
    n, heads = 20, 4
    k = torch.zeros(n, heads, dim, dtype=torch.bfloat16)
    k[:, :, 0] = (torch.rand(n, heads, generator=g) * 8 - 4).bfloat16()
    q = torch.zeros(1, heads, dim, dtype=torch.bfloat16)
    q[0, :, 0] = 1.0
    w = torch.softmax(k[:, :, 0].double() / 4, 0)
    v = torch.stack([_cancelled(w[:, h], torch.randn(n, dim, generator=g).bfloat16())
                     for h in range(heads)], 1)
    cache, table, lengths = _cache(k, v)
    got = cache.attend(q.cuda(), table, lengths, scale=0.25)[0].cpu().double()
    want = (w[:, :, None] * v.double()).sum(0)
    size = (w[:, :, None] * v.double().abs()).sum(0)
    assert (want.abs() < 2.0 ** -22 * size).all()
    R.check(got, want, 2.0 ** -19 * size + R.u(torch.bfloat16) * 2.0 ** -19 * size)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_bf16_rotated_queries(dim):
    """Rotated queries of bf16 pages hold fp32's 24 bits.  Two tokens whose keys pick one member
    each of a pair, 2^11 of it: the scores' difference, 2^11 (y1 - y2), comes out of the weights'
    ratio.  A member is off by the rotation's 2^-20 (|x1| + |x2|) (paged_ref.rotate), a score by
    2^-23 of itself more in fp32 (up to 2^11.5); a member held to 2^-16 would put it off by up to
    2^-5."""
    g = torch.Generator().manual_seed(dim)
    heads = 64
    q = torch.zeros(1, heads, dim, dtype=torch.bfloat16)
    x1 = 1 + torch.rand(heads, generator=g) / 4
    rotary_kw = dict(base=10.0)
    n = 2
    # x2 such that the two members come out close: at angle 1, x1 c - x2 s = x2 c + x1 s
    q[0, :, 0] = x1.bfloat16()
    c, s = math.cos(1), math.sin(1)
    q[0, :, 1] = (q[0, :, 0].float() * (c - s) / (c + s)).bfloat16()
    k = torch.zeros(n, 1, dim, dtype=torch.bfloat16)
    k[0, 0, 0] = k[1, 0, 1] = 2.0 ** 11
    v = torch.zeros(n, 1, dim, dtype=torch.bfloat16)
    v[0], v[1] = 1.0, -1.0
    cache, table, lengths = _cache(k, v, Rotary(2, **rotary_kw))
    got = cache.attend(q.cuda(), table, lengths, scale=0.25)[0].cpu().double()
    y, err = R.rotate(q.float(), torch.tensor([1]), 2, **rotary_kw)
    d = 512 * (y[0, :, 0] - y[0, :, 1])
    off = 512 * (err[0, :, 0] + err[0, :, 1]) + 2.0 ** -21 * 512 * y[0].abs().amax(-1)
    want = torch.tanh(d / 2)[:, None].expand(-1, dim)  # (e^a - e^b) / (e^a + e^b)
    tol = (off / 2)[:, None] * (1 - want ** 2) * 1.01 + (R.u(torch.bfloat16) + 2.0 ** -19) * want.abs() \
        + 2.0 ** -20
    assert (want.abs() < 0.9).any()
    R.check(got, want, tol)
