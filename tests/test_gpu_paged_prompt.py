"""Attention of several new tokens a sequence over its pages (PagedCache.attend with offsets,
adaptq_paged_prompt_device) against the formula in 64 bits: every type, head layout and length at
which it can go wrong, masks of every kind, rows that see nothing, infinities in tokens that are
not seen, pages that are not there, strides, graphs, streams."""
import math
import random

import pytest
import torch

import paged_ref as R
import scores_ref as S

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    globals().update(PagedCache=PagedCache, Rotary=Rotary)


class Case:
    """Queries over a pool: the last new[i] tokens of each sequence."""

    def __init__(self, lengths, new, heads, group, dim, ps, dtype, *, rot=0, seed=0, **kw):
        self.p = S.Pool(lengths, heads, dim, ps, dtype, seed=seed)
        self.new, self.group, self.rot, self.kw = new, group, rot, kw
        self.cache = PagedCache(self.p.k_pages, self.p.v_pages,
                                rotary=Rotary(rot, **kw) if rot else None)
        self.offsets = S.spans(new)
        self.q = self.p.normal(sum(new), heads * group, dim).cuda()
        self.at = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, new)])
        self.of = torch.tensor([i for i, m in enumerate(new) for _ in range(m)])

    def run(self, **kw):
        kw = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        return self.cache.attend(self.q, self.p.table, self.p.lengths, self.offsets, **kw)

    def want(self, *, scale=None, window=None, softcap=None, slopes=None, prefix=None, first=None):
        p, dtype = self.p, self.p.dtype
        q, err = self.q.cpu().double(), None
        if self.rot:
            q, err = R.rotate(self.q.float(), self.at, self.rot, **self.kw)
            q, err = S.rounded(q, err, dtype)
        zero = torch.zeros(len(self.at), dtype=torch.int32)
        outs, tols = [], []
        for i in range(len(self.new)):
            of = self.of == i
            k, v = p.k[i].transpose(0, 1), p.v[i].transpose(0, 1)
            seen = S.sees(k.shape[1], self.at[of], (zero if first is None else first)[of],
                          (zero if prefix is None else prefix)[of], window)
            o, t, _, _ = S.attend(q[of], k, v, seen, self.at[of],
                                  1 / math.sqrt(p.dim) if scale is None else scale, dtype,
                                  softcap=softcap, slopes=slopes,
                                  q_err=None if err is None else err[of],
                                  rough=dtype != torch.float32)
            outs.append(o)
            tols.append(t)
        return torch.cat(outs), torch.cat(tols)

    def check(self, **kw):
        got = self.run(**kw)
        R.check(got, *self.want(**kw))
        return got


# lengths and new tokens: one token, whole prompts, chunks behind a beginning, an empty sequence,
# sequences without new tokens, ends around the tiles of 32, 64 and 128
EDGES = ([1, 31, 32, 33, 64, 65, 200, 0, 129, 300, 77], [1, 31, 32, 33, 64, 65, 1, 0, 129, 127, 0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 104, 128, 160, 192, 256])
@pytest.mark.parametrize("heads,group,ps", [(2, 1, 16), (1, 4, 48)])
def test_lengths(dtype, dim, heads, group, ps):
    Case(*EDGES, heads, group, dim, ps, dtype, seed=dim).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 7), (1, 16), (1, 33), (1, 130), (14, 3)])
def test_groups(dtype, dim, heads, group):
    """Also more query heads a key head than a tile has rows."""
    Case([40, 3, 150], [40, 3, 9], heads, group, dim, 32, dtype, seed=group).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,new", [([5000], [1]), ([4097, 3000], [5, 2]), ([2000] * 3, [40] * 3),
                                         ([9000, 1, 640], [17, 1, 640])])
def test_few_queries_over_many_tokens(dtype, lengths, new):
    """Tiles that are cut over the tokens and joined."""
    c = Case(lengths, new, 2, 4, 128, 64, dtype, seed=len(lengths))
    got = c.check()
    assert torch.equal(c.run(), got)  # equal calls give equal bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [16, 48, 176, 1024])
def test_pages(dtype, ps):
    Case([700, 1500], [700, 300], 2, 2, 64, ps, dtype, seed=ps).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 200, 2 ** 31 - 1])
def test_window(dtype, window):
    Case([0, 1, 33, 100, 640], [0, 1, 33, 50, 640], 2, 3, 64, 16, dtype).check(window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [None, 40])
def test_documents_and_prefixes(dtype, dim, window):
    """Packed documents, some of one token, each with a prefix it sees from both sides."""
    c = Case([500, 260, 90], [500, 200, 90], 2, 2, dim, 16, dtype, seed=dim)
    rng = random.Random(5)
    first, prefix = [], []
    for n, m in zip(c.p.held, c.new):
        start = 0
        while start < n:
            size, pre = rng.choice((1, 2, 63, 64, 65, 130)), rng.choice((0, 1, 17, 70))
            end = min(start + size, n)
            for p in range(max(start, n - m), end):
                first.append(start)
                prefix.append(min(start + pre, end))
            start = end
    first, prefix = (torch.tensor(x, dtype=torch.int32) for x in (first, prefix))
    c.check(first=first, window=window)
    c.check(prefix=prefix, window=window)
    c.check(first=first, prefix=prefix, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_masks(dtype):
    """Every query's own first token and prefix, anywhere: before the tokens, behind them."""
    c = Case([300, 150], [130, 150], 1, 3, 64, 16, dtype)
    g = torch.Generator().manual_seed(1)
    n = len(c.at)
    first = torch.randint(-50, 350, (n,), generator=g).int()
    prefix = torch.randint(-50, 400, (n,), generator=g).int()
    for window in (None, 1, 30):
        c.check(first=first, prefix=prefix, window=window)
    c.check(prefix=torch.full((n,), 2 ** 31 - 1, dtype=torch.int32))  # everything, both ways
    got = c.check(first=torch.full((n,), 2 ** 31 - 1, dtype=torch.int32))
    assert (got == 0).all()  # nothing: zeros


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_caps_and_slopes(dtype, dim):
    c = Case([200, 77, 900], [200, 3, 60], 2, 3, dim, 16, dtype, seed=dim)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(5)] + [0.0])
    c.check(softcap=30.0)
    c.check(softcap=0.5, scale=3.0)  # scores far into the cap
    c.check(slopes=slopes)
    c.check(slopes=-slopes[:6] / 64, window=100)  # a bias towards far tokens
    c.check(softcap=50.0, slopes=slopes, window=33,
            prefix=torch.full((len(c.at),), 20, dtype=torch.int32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1.0, 0.01, -0.5])
def test_scale(dtype, scale):
    Case([40, 200], [40, 100], 2, 2, 64, 16, dtype).check(scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot,interleaved,dim", [(64, False, 64), (64, True, 128), (20, False, 80),
                                                 (6, True, 8), (256, False, 256), (128, False, 128),
                                                 (30, True, 96), (36, False, 72)])
def test_rotated_queries(dtype, rot, interleaved, dim):
    Case([1, 50, 700], [1, 50, 200], 2, 2, dim, 16, dtype, rot=rot, interleaved=interleaved,
         scaling="yarn", factor=4.0, context=512).check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_to_single_queries(dtype):
    """One new token a sequence, through offsets and without: the same formula."""
    c = Case([5, 100, 333], [1, 1, 1], 2, 4, 64, 16, dtype)
    a, b = c.run(softcap=20.0), c.cache.attend(c.q, c.p.table, c.p.lengths, softcap=20.0)
    want, tol = c.want(softcap=20.0)
    R.check(a, want, tol)
    R.check(b, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores in the hundreds, maxima that grow from pass to pass, weights that vanish."""
    c = Case([400], [400], 1, 2, 64, 16, dtype)
    c.p.k[0] = c.p.k[0] * torch.linspace(0.1, 30, 400)[:, None, None].to(dtype)
    c.p.put(0)
    c.check(scale=1.0)
    c.p.k[0] = c.p.k[0].flip(0)
    c.p.put(0)
    c.check(scale=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_infinities_that_are_not_seen(dtype, dim):
    """Infinite and NaN rows reach the queries that see them, and no other."""
    c = Case([300], [300], 2, 2, dim, 16, dtype)
    first = torch.where(torch.arange(300) < 100, 0, 100).int()
    clean = c.run(first=first)
    k, v = c.p.k[0], c.p.v[0]
    v[250, 0, 3] = float("inf")
    v[260, 0, 3] = float("-inf")
    v[40, 0, 5] = float("nan")
    v[99, 1, dim - 1] = float("-inf")
    k[280, 1, 0] = float("nan")
    k[0, 0, 0] = float("inf")  # (its queries' scores are infinite, or NaN)
    c.p.put(0)
    got = c.run(first=first)
    at = torch.arange(300)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[250:, :2, 3] = True
    bad[40:100, :2, 5] = True
    bad[99, 2:, dim - 1] = True
    bad[280:, 2:] = True
    bad[:100, :2] = True
    assert torch.equal(got[~bad], clean[~bad])
    assert (got[250:260, :2, 3] == float("inf")).all()
    assert torch.isnan(got[260:, :2, 3]).all()
    assert (got[99, 2:, dim - 1] == float("-inf")).all()
    assert torch.isnan(got[280:, 2:]).all()
    assert len(at) == 300


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_that_are_seen(dtype):
    """By every query of a tile: as the formula has it."""
    c = Case([600], [20], 1, 2, 64, 16, dtype)
    c.p.v[0][100, 0, 9] = float("inf")
    c.p.v[0][200, 0, 10] = float("nan")
    c.p.put(0)
    got = c.run()
    assert (got[:, :, 9] == float("inf")).all() and torch.isnan(got[:, :, 10]).all()
    assert torch.isfinite(got[:, :, :9]).all() and torch.isfinite(got[:, :, 11:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity(dtype):
    """Only such: a softmax of nothing but zeros, NaN as the formula has it; beside others: no
    weight."""
    c = Case([100, 40], [100, 40], 1, 2, 64, 16, dtype)
    c.q.abs_().add_(0.01)
    c.p.k[0][10:60, :, 0] = -float("inf")
    c.p.k[1][:, :, 0] = -float("inf")
    for i in range(2):
        c.p.put(i)
    got = c.run()
    want, tol = c.want(first=None)
    assert torch.isnan(got[100:]).all()
    c.p.k[0][10:60, :, 0] = 0
    hide = S.sees(100, c.at[:100], torch.zeros(100), torch.zeros(100), None)
    hide[:, 10:60] = False
    out, t, _, _ = S.attend(c.q[:100].cpu().double(), c.p.k[0].transpose(0, 1),
                            c.p.v[0].transpose(0, 1), hide, c.at[:100], 0.125, dtype)
    R.check(got[:100], out, t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_a_page_are_left_out(dtype):
    c = Case([200, 70, 90], [200, 70, 10], 2, 2, 64, 16, dtype)
    t = c.p.table_host
    t[0, 3], t[0, 12] = -1, 10 ** 9  # tokens 48-63 and 192-199
    t[1, :] = 2 ** 31 - 1            # none at all
    c.p.table.copy_(t[:, :c.p.table.shape[1]])
    got = c.run()
    out, tol = [], []
    for i, gone in ((0, [*range(48, 64), *range(192, 200)]), (2, [])):
        of = c.of == i
        n = c.p.held[i]
        seen = S.sees(n, c.at[of], torch.zeros(int(of.sum())), torch.zeros(int(of.sum())), None)
        seen[:, gone] = False
        o, e, _, _ = S.attend(c.q[of.cuda()].cpu().double(), c.p.k[i].transpose(0, 1),
                              c.p.v[i].transpose(0, 1), seen, c.at[of], 0.125, dtype)
        out.append(o)
        tol.append(e)
    R.check(got[(c.of != 1).cuda()], torch.cat(out), torch.cat(tol))
    assert (got[(c.of == 1).cuda()] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_outside_the_offsets_stay(dtype):
    c = Case([50, 30], [20, 30], 2, 2, 64, 16, dtype)
    q = c.p.normal(60, 4, 64).cuda()
    q[5:55] = c.q
    out = torch.full_like(q, 7.0)
    got = c.cache.attend(q, c.p.table, c.p.lengths, c.offsets + 5, out=out)
    assert got is out
    R.check(out[5:55], *c.want())
    assert (out[:5] == 7.0).all() and (out[55:] == 7.0).all()


def test_offsets_and_lengths_that_make_no_sense():
    """Refused by nobody, as they are on the device: outputs are anything, but inside their rows."""
    c = Case([50, 30], [20, 30], 2, 2, 64, 16, torch.bfloat16)
    room = torch.full((70, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[10:60]
    for offsets in ([0, 10 ** 9, -5], [-100, 20, 2 ** 31 - 1], [40, 10, 50], [2 ** 31 - 1] * 3):
        for lengths in ([50, 30], [-5, 10 ** 9], [3, 2 ** 31 - 1]):
            c.cache.attend(c.q, c.p.table, torch.tensor(lengths, dtype=torch.int32).cuda(),
                           torch.tensor(offsets, dtype=torch.int32).cuda(), out=out)
            assert (room[:10] == 7.0).all() and (room[60:] == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_queries_and_outputs(dtype):
    """Queries that are part of a projection, rows off 16 bytes, an output with room around it."""
    c = Case([40, 170], [40, 100], 2, 2, 64, 16, dtype, rot=64)
    q, want = c.q, c.want()
    for pad in (0, 1, 8):
        wide = torch.full((140, 9, 64 + pad), 7.0, dtype=dtype, device="cuda")
        wide[:, 2:6, pad:] = q
        room = torch.full((142, 6, 64 + pad), 5.0, dtype=dtype, device="cuda")
        out = room[1:141, 1:5, pad:]
        got = c.cache.attend(wide[:, 2:6, pad:], c.p.table, c.p.lengths, c.offsets, out=out)
        assert got is out
        R.check(out, *want)
        out.fill_(5.0)
        assert (room == 5.0).all()  # nothing around the rows was written


def test_no_tokens_and_no_sequences():
    c = Case([50, 30], [0, 0], 2, 2, 64, 16, torch.float32)
    assert c.run().shape == (0, 4, 64)
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    out = c.cache.attend(c.q, c.p.table[:0], empty, torch.zeros(1, dtype=torch.int32).cuda())
    assert out.shape == (0, 4, 64)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^31 values a side, its last pages used."""
    pages, heads, ps, dim = 70000, 4, 64, 128
    k, v = (torch.empty(pages, heads, ps, dim, dtype=torch.bfloat16, device="cuda")
            for _ in range(2))
    c = Case([300], [100], heads, 2, dim, ps, torch.bfloat16)
    c.cache = PagedCache(k, v)
    c.p.k_pages, c.p.v_pages = k, v
    c.p.table_host[0, :5] = torch.tensor([69999, 3, 65536, 69998, 40000], dtype=torch.int32)
    c.p.table.copy_(c.p.table_host[:, :c.p.table.shape[1]])
    c.p.put(0)
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dtype):
    """A chunk's append and attention in one graph, whose lengths go on between the replays."""
    c = Case([400, 300], [8, 8], 2, 4, 128, 64, dtype)
    chunk = [c.p.normal(16, 2, 128).cuda() for _ in range(2)]
    lengths = torch.tensor([100, 50], dtype=torch.int32).cuda()
    out = torch.empty_like(c.q)

    def step():
        c.cache.append(*chunk, c.p.table, lengths, c.offsets)
        lengths.add_(c.offsets[1:] - c.offsets[:-1])
        c.cache.attend(c.q, c.p.table, lengths, c.offsets, softcap=10.0, out=out)

    step()
    lengths.copy_(torch.tensor([100, 50], dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lengths.copy_(torch.tensor([100, 50], dtype=torch.int32))
    got = []
    for _ in range(5):
        graph.replay()
        got.append(out.clone())
        (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
    lengths.copy_(torch.tensor([100, 50], dtype=torch.int32))
    for x in got:
        step()
        assert torch.equal(out, x)


def test_streams():
    """A prompt appended on one stream, attended to on another: the cache orders them."""
    c = Case([3000, 2000], [3000, 2000], 4, 4, 128, 64, torch.bfloat16)
    want = c.run()
    k, v = (torch.cat(x).cuda() for x in (c.p.k, c.p.v))
    zero = torch.zeros_like(c.p.lengths)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        c.p.k_pages.fill_(float("nan"))
        c.p.v_pages.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            c.cache.append(k, v, c.p.table, zero, c.offsets)
        with torch.cuda.stream(b):
            got = c.run()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals():
    c = Case([50, 30], [20, 30], 2, 2, 64, 16, torch.bfloat16)
    q, table, lengths, at = c.q, c.p.table, c.p.lengths, c.offsets
    run = c.cache.attend
    for kw in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=float("nan")), dict(window=0),
               dict(scale=0.0), dict(slopes=torch.ones(3, device="cuda")),
               dict(slopes=torch.ones(4, device="cuda", dtype=torch.float16)),
               dict(slopes=torch.ones(4)), dict(prefix=torch.ones(49, dtype=torch.int32).cuda()),
               dict(first=torch.ones(50, device="cuda")),
               dict(first=torch.ones(100, dtype=torch.int32).cuda()[::2]),
               dict(weights=torch.zeros(2, 2, 64, device="cuda")), dict(out=torch.empty_like(q[1:]))):
        with pytest.raises((ValueError, TypeError)):
            run(q, table, lengths, at, **kw)
    for bad in (at[:2], at.long(), at.cpu()):
        with pytest.raises((ValueError, TypeError)):
            run(q, table, lengths, bad)
    with pytest.raises(RuntimeError):
        run(q[:, :3], table, lengths, at)  # not a multiple of the key heads
    with pytest.raises(RuntimeError):
        run(q, table, lengths, at, out=q)  # an output over its input
    with pytest.raises(RuntimeError):
        run(q, table, lengths, at, softcap=1e38 * 10)
