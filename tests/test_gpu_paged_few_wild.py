"""Infinities among the values of a prompt of few rows (which the single-token kernel takes), at
every weight that a token can have, in units that all rows see and in those that some see."""
import pytest
import torch

import paged_ref as R
import test_gpu_paged_prompt as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    P.PagedCache, P.Rotary = PagedCache, Rotary


@pytest.mark.parametrize("dtype", P.DTYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("n,new,kw", [(2000, 3, {}), (2000, 8, dict(softcap=1e4)), (30000, 4, {}),
                                      (2000, 5, dict(window=1990))])
def test_of_any_weight(dtype, dim, n, new, kw):
    """From e^0 down to e^-90, and of two signs: the infinity, or NaN where both meet; other
    channels as without them."""
    c = P.Case([n], [new], 1, 2, dim, 16, dtype)
    scores = -(torch.arange(n) % 91).float()
    c.q.fill_(1.0)  # every query's score of token t: scores[t]
    c.p.k[0][:] = (scores / dim).to(dtype)[:, None, None]
    c.p.put(0)
    kw = dict(scale=1.0, **kw)
    clean = c.run(**kw)
    for i in range(40):
        c.p.v[0][50 + (37 * i) % 1600, 0, i] = float("inf") if i % 2 else -float("inf")
    c.p.v[0][63, 0, 50], c.p.v[0][700, 0, 50] = float("inf"), -float("inf")
    c.p.v[0][n - 2, 0, 60] = float("inf")  # that the first queries do not see
    c.p.put(0)
    got = c.run(**kw)
    for i in range(40):
        assert (got[:, :, i] == (float("inf") if i % 2 else -float("inf"))).all(), i
    assert torch.isnan(got[:, :, 50]).all()
    assert (got[-2:, :, 60] == float("inf")).all()
    assert torch.equal(got[:-2, :, 60], clean[:-2, :, 60])
    rest = [i for i in range(40, dim) if i not in (50, 60)]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])
    R.check(got[:, :, rest], *(x[:, :, rest] for x in c.want(**kw)))


@pytest.mark.parametrize("dtype", P.DTYPES)
@pytest.mark.parametrize("n", [700, 30000])
def test_in_a_part_of_no_weight(dtype, n):
    """All of a wave's or a piece's tokens weigh e^-100 beside the others', and one of them is
    infinite."""
    c = P.Case([n], [4], 1, 2, 64, 16, dtype)
    scores = torch.zeros(n)
    scores[:n * 3 // 4] = -100.0
    c.q.fill_(1.0)
    c.p.k[0][:] = (scores / 8).to(dtype)[:, None, None]
    c.p.put(0)
    clean = c.check()
    c.p.v[0][40, 0, 3] = float("inf")
    c.p.v[0][n * 3 // 4 - 70, 0, 4] = -float("inf")
    c.p.v[0][n // 2, 0, 5] = float("nan")
    c.p.put(0)
    got = c.run()
    assert (got[:, :, 3] == float("inf")).all() and (got[:, :, 4] == -float("inf")).all()
    assert torch.isnan(got[:, :, 5]).all()
    rest = [0, 1, 2, *range(6, 64)]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])
