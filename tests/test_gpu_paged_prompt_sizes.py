"""Prompts at the last positions that a sequence can have: tokens end at 2^31 - 33."""
import math

import pytest
import torch

import paged_ref as R
import scores_ref as S

pytestmark = pytest.mark.gpu
LAST = 2 ** 31 - 32  # tokens at the most


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    globals().update(PagedCache=PagedCache)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [2 ** 31 - 65, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 33, 2 ** 31 - 32,
                               2 ** 31 - 20, 2 ** 31 - 1])
@pytest.mark.parametrize("heads,sequences", [(1, 1), (8, 64)])
def test_the_last_positions(dtype, n, heads, sequences):
    """Windows, first tokens that a window keeps, documents; tiles that are cut (one sequence) and
    whole ones; an infinity in the last unit that some queries do not see."""
    page, dim, new = 65536, 64, 40
    g = torch.Generator("cuda").manual_seed(n & 255)
    k, v = (torch.randn(2, heads, page, dim, generator=g, device="cuda").to(dtype)
            for _ in range(2))
    q = torch.randn(sequences * new, 2 * heads, dim, generator=g, device="cuda").to(dtype)
    table = torch.zeros(sequences, 32768, dtype=torch.int32)
    table[:, -1] = 1
    lengths, offsets = torch.full((sequences,), n, dtype=torch.int32).cuda(), S.spans([new] * sequences)
    at = torch.arange(n - new, n)
    # the tokens that count: the first 16, and the last 400
    start = LAST - 400
    t = torch.cat((torch.arange(16), torch.arange(start, LAST)))
    slots = torch.arange(start, LAST) - (2 ** 31 - page)
    for window, first, prefix in ((100, None, None), (70, None, 5), (None, start + 101, None),
                                  (33, start + 50, 3)):
        for wild in (False, True):
            vv = v.clone()
            inside = min(n, LAST) - 20  # (of position n - 20 or before: some queries see it not)
            if wild and n <= LAST:
                vv[1, :, inside - (2 ** 31 - page), 7] = float("inf")
            cache = PagedCache(k, vv)
            kw = {name: None if x is None else torch.full((q.shape[0],), x, dtype=torch.int32).cuda()
                  for name, x in (("first", first), ("prefix", prefix))}
            got = cache.attend(q, table.cuda(), lengths, offsets, window=window, **kw)[-new:].cpu()
            seen = (t[None] <= at[:, None]) & (t[None] < n)
            if window:
                seen &= t[None] > at[:, None] - window
            if prefix:
                seen |= t[None] < prefix
            if first:
                seen &= t[None] >= first
            for h in {0, heads - 1}:
                kk, vh = (torch.cat((x[0, h, :16].cpu(), x[1, h].cpu()[slots]))[None]
                          for x in (k, v))
                o, tol, _, _ = S.attend(q[-new:, 2 * h:2 * h + 2].cpu().double(), kk, vh, seen, at,
                                        1 / math.sqrt(dim), dtype)
                x = got[:, 2 * h:2 * h + 2]
                if wild and n <= LAST:
                    sees = (at >= inside) & (at - inside < (window or 10 ** 9))
                    assert (x[sees, :, 7] == float("inf")).all() and sees.any() and not sees.all()
                    x = torch.where((sees[:, None, None]) & (torch.arange(dim) == 7), o.to(x.dtype), x)
                R.check(x, o, tol, f"window {window} first {first} prefix {prefix} head {h}")
