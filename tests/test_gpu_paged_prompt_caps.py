"""Prompts whose scores are capped by more than the scores themselves come to: a cap of any size
leaves scores that are small beside it as they are."""
import math

import pytest
import torch

import paged_ref as R
import scores_ref as S
import test_gpu_paged_prompt as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    P.PagedCache, P.Rotary = PagedCache, Rotary


def want(c, cap):
    """Above 64 the tanh is within 2^-21 of its value, whatever the cap: S.attend's tolerance
    without `rough`.  (scale / cap is a normal number, or one of 22 bits at the least, for caps up
    to 1e37.)"""
    outs, tols = [], []
    for i in range(len(c.new)):
        of = c.of == i
        k, v = c.p.k[i].transpose(0, 1), c.p.v[i].transpose(0, 1)
        none = torch.zeros(int(of.sum()))
        seen = S.sees(k.shape[1], c.at[of], none, none, None)
        o, t, _, _ = S.attend(c.q.cpu().double()[of], k, v, seen, c.at[of],
                              1 / math.sqrt(c.p.dim), c.p.dtype, softcap=cap)
        outs.append(o)
        tols.append(t)
    return torch.cat(outs), torch.cat(tols)


@pytest.mark.parametrize("dtype", P.DTYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("cap", [65.0, 1e4, 1e7, 1e9, 1e20, 1e37])
def test_large_caps(dtype, dim, cap):
    c = P.Case([200, 77, 900], [200, 3, 60], 2, 3, dim, 16, dtype, seed=dim)
    R.check(c.run(softcap=cap), *want(c, cap), f"cap {cap}")


@pytest.mark.parametrize("dtype", P.DTYPES)
def test_the_number_of_new_tokens_does_not_change_the_cap(dtype):
    """One call of many rows, one of few and one of single queries: the same formula."""
    c = P.Case([300], [40], 2, 4, 64, 16, dtype)
    o, tol = want(c, 1e8)
    R.check(c.run(softcap=1e8), o, tol, "many")
    for m in (3, 1):
        last = c.cache.attend(c.q[-m:], c.p.table, c.p.lengths, S.spans([m]), softcap=1e8)
        R.check(last, o[-m:], tol[-m:], str(m))
    one = c.cache.attend(c.q[-1:], c.p.table, c.p.lengths, softcap=1e8)
    R.check(one, o[-1:], tol[-1:], "one")
