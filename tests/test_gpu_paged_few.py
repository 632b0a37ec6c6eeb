"""Prompts of a few rows a key head and sequence (draft tokens, short chunks), which the
single-token kernel takes, against the formula in 64 bits: every type, head size and number of
rows, lengths that differ, many sequences, masks, rows that see nothing, infinities in tokens that
some rows do not see, graphs whose offsets move on."""
import pytest
import torch

import paged_ref as R
import scores_ref as S
import test_gpu_paged_prompt as P

pytestmark = pytest.mark.gpu
DTYPES = P.DTYPES


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    P.PagedCache, P.Rotary = PagedCache, Rotary


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 104, 128, 160, 192, 256])
@pytest.mark.parametrize("group,new", [(1, [1, 7, 16, 3, 0, 16, 5]), (4, [4, 4, 1, 2, 0, 4, 3]),
                                       (16, [1, 1, 1, 1, 0, 1, 1]), (5, [2, 3, 3, 3, 0, 3, 3])])
def test_lengths(dtype, dim, group, new):
    """One tile and a little more (rows of a query in two tiles), around the units' ends."""
    lengths = [2, 16, 33, 64, 100, 700, 1025]
    c = P.Case(lengths, new, 2, group, dim, 16, dtype, seed=dim)
    got = c.check()
    assert torch.equal(c.run(), got)
    c.check(window=9)
    c.check(softcap=3.0, scale=0.5, slopes=torch.linspace(-0.01, 0.5, 2 * group))
    c.check(prefix=torch.tensor([(37 * i) % 90 - 9 for i in range(len(c.at))], dtype=torch.int32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_sequence_has_nearly_all_of_them(dtype):
    """The choice is made by the average: others have one query, or none."""
    c = P.Case([3, 900, 50, 1, 800, 20], [0, 19, 1, 1, 0, 1], 2, 4, 128, 32, dtype)
    c.check()
    c.check(window=500, slopes=torch.ones(8) / 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    """More than one look at 64 lengths; runs of sequences without queries."""
    lengths = [(i * 37) % 150 for i in range(200)]
    new = [0 if 60 < i < 140 else min(n, i % 5) for i, n in enumerate(lengths)]
    c = P.Case(lengths, new, 2, 4, 64, 16, dtype)
    c.check()
    c.check(window=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,ps", [(1, 16), (8, 64)])
def test_long(dtype, heads, ps):
    """Segments that are cut and joined, in groups too; windows that leave most of them out."""
    c = P.Case([20000, 300, 9000], [4, 3, 4], heads, 4, 128, ps, dtype)
    got = c.check()
    assert torch.equal(c.run(), got)
    c.check(window=4500)
    c.check(prefix=torch.tensor([20000, 0, 19999, 7, 0, 290, 300] + [8999] * 4, dtype=torch.int32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot,interleaved,dim", [(64, False, 64), (64, True, 128), (20, False, 80),
                                                 (256, False, 256)])
def test_rotated(dtype, rot, interleaved, dim):
    P.Case([3, 50, 700], [3, 4, 4], 2, 4, dim, 16, dtype, rot=rot, interleaved=interleaved).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
@pytest.mark.parametrize("n", [300, 4000])
def test_infinities_that_some_do_not_see(dtype, dim, n):
    """Among the newest tokens: they reach the queries from their own on, in both signs and as
    NaN, in every key head's own rows."""
    c = P.Case([n, n], [7, 7], 2, 2, dim, 16, dtype)
    clean = c.run()
    k, v = c.p.k[0], c.p.v[0]
    v[n - 3, 0, 3] = float("inf")
    v[n - 2, 0, 3] = float("-inf")
    v[n - 4, 1, dim - 1] = float("-inf")
    v[n - 1, 1, 0] = float("nan")
    k[n - 2, 1, 5] = float("nan")
    c.p.put(0)
    bad = torch.zeros_like(clean, dtype=torch.bool)
    bad[4:7, :2, 3] = True
    bad[3:7, 2:, dim - 1] = True
    bad[5:7, 2:] = True
    for got in (c.run(), c.run(window=n)):
        assert torch.equal(got[~bad], clean[~bad])
        assert (got[4, :2, 3] == float("inf")).all()
        assert torch.isnan(got[5:7, :2, 3]).all() and torch.isnan(got[5:7, 2:]).all()
        assert (got[3:5, 2:, dim - 1] == float("-inf")).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_behind_a_window(dtype):
    """The first query sees one, the later ones no more; one that nobody sees; one in a row whose
    page stands beside one that is not there."""
    c = P.Case([200], [5], 1, 3, 64, 16, dtype)
    clean = c.run(window=100)
    c.p.v[0][96, 0, 2] = float("inf")  # queries at 195 to 199 see from 96 to 100 on
    c.p.v[0][95, 0, 1] = float("nan")
    c.p.k[0][95, 0, 1] = float("nan")
    c.p.put(0)
    got = c.run(window=100)
    assert (got[0, :, 2] == float("inf")).all()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :, 2] = True
    assert torch.equal(got[~bad], clean[~bad])
    c.p.v[0][150, 0, 7] = float("-inf")  # seen by all, in a unit whose other block has no page
    c.p.put(0)
    c.p.table_host[0, 8] = -1
    c.p.table.copy_(c.p.table_host[:, :c.p.table.shape[1]])
    assert (c.run(window=100)[:, :, 7] == float("-inf")).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_that_see_nothing(dtype):
    """More queries than tokens: those at negative positions, and of empty sequences, get zeros."""
    c = P.Case([3, 5, 40], [3, 4, 4], 2, 2, 64, 16, dtype)
    want, tol = c.want()
    c.p.lengths.copy_(torch.tensor([1, 0, 40], dtype=torch.int32))
    got = c.run()
    assert (got[:2] == 0).all() and (got[3:7] == 0).all()
    first = c.p.v[0][0].cuda().repeat_interleave(2, 0)
    assert torch.equal(got[2], first)  # one token: its value
    R.check(got[7:], want[7:], tol[7:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_while_offsets_move(dtype):
    """One graph, whose sequences' queries and lengths change between the replays."""
    c = P.Case([500, 400, 60], [4, 4, 4], 2, 4, 128, 16, dtype)
    out = torch.empty_like(c.q)
    c.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.cache.attend(c.q, c.p.table, c.p.lengths, c.offsets, softcap=9.0, out=out)
    for lengths, new in (([500, 400, 60], [4, 4, 4]), ([17, 400, 60], [0, 12, 0]),
                         ([500, 1, 60], [5, 1, 6]), ([500, 400, 60], [4, 4, 4])):
        c.p.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        c.offsets.copy_(S.spans(new))
        graph.replay()
        got = out.clone()
        (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
        assert torch.equal(got, c.run(softcap=9.0))


def test_beside_single_tokens():
    """Calls of both kinds in turn, which share the cache's workspace."""
    c = P.Case([9000, 4000], [4, 4], 8, 4, 128, 64, torch.bfloat16)
    many, one = c.run(), c.cache.attend(c.q[:2], c.p.table, c.p.lengths)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(a):
            x = c.run()
        with torch.cuda.stream(b):
            y = c.cache.attend(c.q[:2], c.p.table, c.p.lengths)
        torch.cuda.synchronize()
        assert torch.equal(x, many) and torch.equal(y, one)
