"""Infinities and NaN among the values that every query of a prompt's tile sees, at every weight
that a token can have; values near the end of fp32's range."""
import math

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


def rising(c, scores):
    """Every query's score of token t becomes scores[t] (times 1 / 8 of 64 ones)."""
    c.q.fill_(1.0)
    c.p.k[0][:] = (scores / 8).to(c.p.dtype)[:, None, None]


@pytest.mark.parametrize("dtype", P.DTYPES)
@pytest.mark.parametrize("kw", [dict(softcap=30.0), dict(slopes=torch.zeros(2)), {}])
def test_of_the_largest_weight(dtype, kw):
    """It is 1, which one number holds: the other is 0, and 0 times an infinity is NaN."""
    c = P.Case([600], [20], 1, 2, 64, 16, dtype)
    scores = torch.zeros(600)
    scores[100] = 24.0
    rising(c, scores)
    c.p.v[0][100, 0, 9] = float("inf")
    c.p.v[0][100, 0, 11] = -float("inf")
    c.p.v[0][130, 0, 10] = float("nan")
    c.p.put(0)
    got = c.run(**kw)
    assert (got[:, :, 9] == float("inf")).all() and (got[:, :, 11] == -float("inf")).all()
    assert torch.isnan(got[:, :, 10]).all()
    keep = [i for i in range(64) if i not in (9, 10, 11)]
    assert torch.isfinite(got[:, :, keep]).all()


@pytest.mark.parametrize("dtype", P.DTYPES)
@pytest.mark.parametrize("n,new", [(2000, 20), (2000, 300), (9000, 20)])
def test_of_any_weight(dtype, n, new):
    """From e^0 down to e^-90, and of two signs: the infinity, or NaN where both meet; other
    channels and queries before the infinities as without them."""
    c = P.Case([n], [new], 1, 2, 64, 16, dtype)
    scores = -(torch.arange(n) % 91).float()
    rising(c, scores)
    c.p.put(0)
    clean = c.run()
    for i in range(40):
        c.p.v[0][(37 * i) % 1600, 0, i] = float("inf") if i % 2 else -float("inf")
    c.p.v[0][3, 0, 50], c.p.v[0][700, 0, 50] = float("inf"), -float("inf")
    c.p.v[0][n - 9, 0, 60] = float("inf")  # that the first queries do not see
    c.p.put(0)
    got = c.run()
    for i in range(40):
        assert (got[:, :, i] == (float("inf") if i % 2 else -float("inf"))).all(), i
    assert torch.isnan(got[:, :, 50]).all()
    assert (got[-9:, :, 60] == float("inf")).all()
    assert torch.equal(got[:-9, :, 60], clean[:-9, :, 60])
    rest = [i for i in range(40, 64) if i not in (50, 60)]
    R.check(got[:, :, rest], *(x[:, :, rest] for x in c.want()))
    assert torch.equal(c.run().nan_to_num(7.0), got.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", P.DTYPES)
def test_in_a_piece_of_no_weight(dtype):
    """A tile that is cut: all of the first piece's tokens weigh e^-100 beside the others', and one
    of them is infinite."""
    c = P.Case([6000], [20], 1, 2, 64, 16, dtype)
    scores = torch.zeros(6000)
    scores[:3000] = -100.0
    rising(c, scores)
    c.p.put(0)
    clean = c.check()
    c.p.v[0][40, 0, 3] = float("inf")
    c.p.v[0][2990, 0, 4] = -float("inf")
    c.p.v[0][1500, 0, 5] = float("nan")
    c.p.put(0)
    got = c.run()
    assert (got[:, :, 3] == float("inf")).all() and (got[:, :, 4] == -float("inf")).all()
    assert torch.isnan(got[:, :, 5]).all()
    rest = [0, 1, 2, *range(6, 64)]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,new", [(500, 30), (6000, 20)])
def test_values_near_the_end_of_fp32(dtype, n, new):
    """A maximum that grows by less than 2^8 a pass, and a value of 2^126 at its top: the formula
    is finite, so is the output."""
    c = P.Case([n], [new], 1, 2, 64, 16, dtype)
    at = torch.arange(n) % 128  # (where the pieces of a cut tile begin, of four passes or more)
    scores = (at >= 32) * 2.0 + (at >= 64) * 2.0
    scores[456] = 5.0
    rising(c, scores)
    c.p.v[0].zero_()
    c.p.v[0][456, 0, 5] = 2.0 ** 126
    c.p.v[0][457, 0, 6] = -2.0 ** 126
    c.p.put(0)
    want, tol = c.want()
    assert want.abs().max() > 2.0 ** 110
    R.check(c.run(), want, tol)


def test_prompts_of_all_types_of_trouble_in_one_batch():
    """A sequence with infinities beside others without: theirs are the same bits as alone."""
    c = P.Case([700, 500], [64, 64], 2, 2, 128, 64, torch.bfloat16)
    clean = c.run()
    c.p.v[0][5, :, 3] = float("inf")
    c.p.k[0][5, :] = c.p.k[0][5, :] * 40
    c.p.put(0)
    got = c.run()
    assert torch.equal(got[64:], clean[64:])
    assert math.isinf(got[0, 0, 3].item()) and torch.isfinite(got[:64, :, 4:]).all()


def test_nan_queries():
    """One query that is NaN beside others that are not."""
    c = P.Case([400], [40], 1, 2, 64, 16, torch.bfloat16)
    clean = c.run()
    c.q[7, 1] = float("nan")
    got = c.run()
    assert torch.isnan(got[7, 1]).all()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[7, 1] = True
    assert torch.equal(got[~bad], clean[~bad])
