"""What the paged attention holds rotated fp16 queries to, whatever their size, against the
formula in 64 bits."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


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
