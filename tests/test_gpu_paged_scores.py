"""Attention of one new token a sequence with scores of its own (caps, biases, prefixes, first
tokens) and the weights it adds up, against the formula in 64 bits; as one step with the append;
and through the C entries."""
import ctypes as C
import math

import pytest
import torch

import paged_ref as R
import scores_ref as S
from adaptq_amd import _lib

pytestmark = pytest.mark.gpu
L = _lib.lib
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    globals().update(PagedCache=PagedCache, Rotary=Rotary)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 700, 0]


class Case:
    def __init__(self, lengths, heads, group, dim, ps, dtype, *, rot=0, seed=0):
        self.p = S.Pool(lengths, heads, dim, ps, dtype, seed=seed, extra=1)
        self.rot = rot
        self.cache = PagedCache(self.p.k_pages, self.p.v_pages, rotary=Rotary(rot) if rot else None)
        self.q = self.p.normal(len(lengths), heads * group, dim).cuda()

    def weights(self, value=0.0, more=0):
        p = self.p
        w = torch.rand(len(p.held), p.heads, p.table.shape[1] * p.ps + more, generator=p.g)
        return (w * value).cuda()

    def want(self, *, scale=None, window=None, softcap=None, slopes=None, prefix=None, first=None,
             weights=None):
        p = self.p
        outs, tols, sums, sum_tols = [], [], [], []
        for i, n in enumerate(p.held):
            q, err = self.q[i:i + 1].cpu().double(), None
            if self.rot and n:
                q, err = R.rotate(self.q[i:i + 1].float(), torch.tensor([n - 1]), self.rot)
            at = torch.tensor([n - 1])
            seen = S.sees(n, at, torch.zeros(1) if first is None else first[i:i + 1],
                          torch.zeros(1) if prefix is None else prefix[i:i + 1], window)
            o, t, m, mt = S.attend(q, p.k[i].transpose(0, 1), p.v[i].transpose(0, 1), seen, at,
                                   1 / math.sqrt(p.dim) if scale is None else scale, p.dtype,
                                   softcap=softcap, slopes=slopes, q_err=err)
            outs.append(o)
            tols.append(t)
            if weights is not None:
                x = weights[i].cpu().double()
                x[:, :n] += m
                e = torch.zeros_like(x)
                e[:, :n] = mt + 2.0 ** -23 * x[:, :n].abs()
                sums.append(x)
                sum_tols.append(e)
        if weights is None:
            return torch.cat(outs), torch.cat(tols)
        return torch.cat(outs), torch.cat(tols), torch.stack(sums), torch.stack(sum_tols)

    def check(self, weights=None, **kw):
        want = self.want(weights=weights, **kw)
        gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        if weights is None:
            got = self.cache.attend(self.q, self.p.table, self.p.lengths, **gpu)
            R.check(got, *want)
            return got
        w = weights.clone()
        got = self.cache.attend(self.q, self.p.table, self.p.lengths, weights=w, **gpu)
        R.check(got, *want[:2])
        R.check(w, *want[2:], "weights")
        return got, w


def some(n, lo, hi, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi, (n,), generator=g).int()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 64, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("heads,group,ps", [(2, 1, 16), (1, 5, 48)])
def test_lengths(dtype, dim, heads, group, ps):
    c = Case(EDGES, heads, group, dim, ps, dtype, seed=dim)
    slopes = torch.linspace(-0.01, 0.5, heads * group)
    c.check(softcap=20.0)
    c.check(slopes=slopes)
    c.check(softcap=50.0, slopes=slopes, weights=c.weights(1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 7), (1, 16), (2, 17), (1, 40), (14, 3)])
def test_groups(dtype, heads, group):
    c = Case([5, 100, 0, 333], heads, group, 64, 32, dtype, seed=group)
    c.check(softcap=10.0, slopes=torch.rand(heads * group), weights=c.weights())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [None, 1, 2, 31, 33, 100, 500, 2 ** 31 - 1])
def test_masks(dtype, window):
    """First tokens and prefixes anywhere, with and without a hole between prefix and window."""
    lengths = [0, 1, 33, 100, 101, 640, 2000, 1999]
    c = Case(lengths, 2, 3, 64, 16, dtype)
    n = len(lengths)
    for first, prefix in ((some(n, -3, 40), None), (None, some(n, -3, 60, 1)),
                          (some(n, 0, 30, 2), some(n, 0, 300, 3)), (some(n, 0, 3000, 4), None),
                          (some(n, 0, 3000, 5), some(n, 0, 3000, 6)),
                          (torch.full((n,), 2 ** 31 - 1, dtype=torch.int32), None),
                          (None, torch.full((n,), 2 ** 31 - 1, dtype=torch.int32))):
        kw = {k: x for k, x in (("first", first), ("prefix", prefix)) if x is not None}
        c.check(window=window, weights=c.weights(0.5), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,ps", [([20000], 64), ([9000, 1, 700], 16), ([5000, 4097], 256)])
def test_long(dtype, lengths, ps):
    """Cut over their tokens and joined; a hole of many pages."""
    c = Case(lengths, 2, 4, 128, ps, dtype)
    c.check(softcap=30.0, weights=c.weights())
    prefix = torch.full((len(lengths),), 70, dtype=torch.int32)
    c.check(window=1000, prefix=prefix, weights=c.weights())
    got, w = c.check(window=3000, prefix=prefix, softcap=5.0, weights=c.weights())
    again, w2 = c.check(window=3000, prefix=prefix, softcap=5.0, weights=c.weights())
    assert torch.equal(got, again) and torch.equal(w, w2)  # equal calls give equal bits


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotated(dtype):
    c = Case([1, 50, 700, 0], 2, 4, 128, 16, dtype, rot=128)
    c.check(softcap=30.0, slopes=torch.rand(8), weights=c.weights())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1.0, -0.5, 0.01])
def test_scale_and_cap(dtype, scale):
    c = Case([40, 200], 2, 2, 64, 16, dtype)
    c.check(scale=scale, softcap=2.0)
    c.check(scale=scale, weights=c.weights())


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_sum_to_the_query_heads(dtype):
    c = Case([700, 33, 0, 4000], 2, 4, 64, 64, dtype)
    w = c.weights(more=5)
    c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w)
    total = w.double().sum(2).cpu()
    assert (total[[0, 1, 3]] - 4).abs().max() < 1e-4 and (total[2] == 0).all()
    for i, n in enumerate(c.p.held):
        assert (w[i, :, n:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_weights(dtype):
    """A part of a larger tensor: what lies around it stays."""
    c = Case([100, 300], 2, 2, 64, 16, dtype)
    tokens = c.p.table.shape[1] * 16
    room = torch.full((3, 4, tokens + 7), 5.0, device="cuda")
    w = room[1:, 1:3, 3:3 + tokens]
    want = c.want(weights=w)
    c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w)
    R.check(w, *want[2:], "weights")
    w.fill_(5.0)
    assert (room == 5.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_that_are_not_seen(dtype):
    c = Case([100, 200], 2, 2, 64, 16, dtype)
    kw = dict(window=20, prefix=torch.tensor([5, 5], dtype=torch.int32).cuda(),
              first=torch.tensor([2, 0], dtype=torch.int32).cuda())
    w = c.weights()
    clean = c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w, **kw)
    for x in (c.p.k, c.p.v):
        x[0][0] = float("nan")
        x[0][6:79] = float("inf")
        x[1][5:180] = float("nan")
    c.p.put(0)
    c.p.put(1)
    w2 = c.weights()
    assert torch.equal(c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w2, **kw), clean)
    assert torch.equal(w, w2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_not_there(dtype):
    c = Case([200, 70], 2, 2, 64, 16, dtype)
    c.p.table_host[0, 3], c.p.table_host[1, :] = -1, 2 ** 31 - 1
    c.p.table.copy_(c.p.table_host[:, :c.p.table.shape[1]])
    w = c.weights()
    got = c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w, softcap=9.0)
    seen = S.sees(200, torch.tensor([199]), torch.zeros(1), torch.zeros(1), None)
    seen[:, 48:64] = False
    o, t, m, mt = S.attend(c.q[:1].cpu().double(), c.p.k[0].transpose(0, 1),
                           c.p.v[0].transpose(0, 1), seen, torch.tensor([199]), 0.125, dtype,
                           softcap=9.0)
    R.check(got[:1], o, t)
    R.check(w[0, :, :200], m, mt + 2.0 ** -23 * m)
    assert (got[1] == 0).all() and (w[1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [None, 100, 10 ** 6])
def test_step(dtype, first):
    """Append and attention in one: the pages and outputs of the two calls, also where the new
    token is itself not seen."""
    c = Case([0, 1, 31, 64, 100, 700], 2, 3, 64, 16, dtype, rot=64)
    n = len(c.p.held)
    k, v = c.p.normal(n, 2, 64).cuda(), c.p.normal(n, 2, 64).cuda()
    kw = dict(window=50, softcap=20.0, prefix=torch.full((n,), 9, dtype=torch.int32).cuda())
    if first is not None:
        kw["first"] = torch.full((n,), first, dtype=torch.int32).cuda()
    other = PagedCache(c.p.k_pages.clone(), c.p.v_pages.clone(), rotary=Rotary(64))
    w, w2 = c.weights(), c.weights()
    got = c.cache.step(c.q, k, v, c.p.table, c.p.lengths, weights=w, **kw)
    other.append(k, v, c.p.table, c.p.lengths)
    want = other.attend(c.q, c.p.table, c.p.lengths + 1, weights=w2, **kw)
    assert torch.equal(got, want) and torch.equal(w, w2)
    for a, b in ((c.cache.k_pages, other.k_pages), (c.cache.v_pages, other.v_pages)):
        assert torch.equal(a.nan_to_num(3.0), b.nan_to_num(3.0))


def test_captured_and_replayed():
    """Steps whose weights add up, in one graph."""
    c = Case([100, 333], 2, 4, 128, 64, torch.bfloat16)
    k, v = c.p.normal(2, 2, 128).cuda(), c.p.normal(2, 2, 128).cuda()
    start = torch.tensor([50, 100], dtype=torch.int32).cuda()
    lengths, w, out = start.clone(), c.weights(), torch.empty_like(c.q)

    def step():
        c.cache.step(c.q, k, v, c.p.table, lengths, weights=w, softcap=20.0, out=out)
        lengths.add_(1)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lengths.copy_(start)
    w.zero_()
    got = []
    for _ in range(5):
        graph.replay()
        got.append((out.clone(), w.clone()))
        (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
    lengths.copy_(start)
    w.zero_()
    for x, y in got:
        step()
        assert torch.equal(out, x) and torch.equal(w, y)


def test_versions_rise():
    c = Case([10], 2, 2, 64, 16, torch.float16)
    w = c.weights()
    before = w._version
    c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w)
    assert w._version > before


def test_refusals():
    c = Case([10, 20], 2, 2, 64, 16, torch.float16)
    tokens = c.p.table.shape[1] * 16
    good = torch.zeros(2, 2, tokens, device="cuda")
    for w in (good[:1], good[:, :1], good[:, :, 1:], good.double(), good.cpu(),
              torch.zeros(2, 2, 2 * tokens, device="cuda")[:, :, ::2]):
        with pytest.raises(ValueError):
            c.cache.attend(c.q, c.p.table, c.p.lengths, weights=w)
    with pytest.raises(RuntimeError):  # rows over each other
        c.cache.attend(c.q, c.p.table, c.p.lengths, weights=good[:, :1].expand(2, 2, tokens))
    pages = c.p.k_pages.flatten().view(torch.float32)[:4 * tokens].view(2, 2, tokens)
    room = torch.zeros(2 ** 12, device="cuda")
    over = room[:4 * tokens].view(2, 2, tokens)
    rows = room.view(torch.float16)[128:640].view(2, 4, 64)
    for w, q, out in ((pages, c.q, None), (over, rows, None), (over, c.q, rows)):  # over the rows
        with pytest.raises(RuntimeError, match="overlap"):
            c.cache.attend(q, c.p.table, c.p.lengths, weights=w, out=out)
    with pytest.raises(RuntimeError, match="overlap"):
        c.cache.step(c.q, rows[:, :2], c.q[:, 2:], c.p.table, c.p.lengths, weights=over)
    for kw in (dict(softcap=0.0), dict(slopes=torch.zeros(5, device="cuda")),
               dict(first=torch.zeros(2, device="cuda")),
               dict(prefix=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            c.cache.attend(c.q, c.p.table, c.p.lengths, **kw)
        with pytest.raises(ValueError):
            c.cache.step(c.q, c.q[:, :2], c.q[:, :2], c.p.table, c.p.lengths, **kw)


def test_c_entries():
    """The C entries with byte strides of their own, and what they refuse."""
    c = Case([40, 200], 2, 2, 64, 16, torch.float32)
    h = L.adaptq_paged_create(c.p.k_pages.data_ptr(), c.p.v_pages.data_ptr(), c.p.pages, 16, 2, 64, 0,
                              None)
    assert h
    out, w = torch.empty_like(c.q), c.weights()
    need = L.adaptq_paged_weights_workspace(h, 4, 2, c.p.table.shape[1])
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    slopes = torch.rand(4).cuda()
    sc = _lib.Scores(20.0, 0, slopes.data_ptr(), None, None)
    stride = c.p.table.stride(0)

    def attend(scale=0.0, sc=sc, w=w, need=need, space=space):
        return L.adaptq_paged_attend_scores_device(
            h, c.q.data_ptr(), out.data_ptr(), 4, 256, 1024, 256, 1024, c.p.table.data_ptr(),
            c.p.table.shape[1], stride, c.p.lengths.data_ptr(), 2, scale, sc and C.byref(sc),
            w.data_ptr() if w is not None else None, 4 * w.stride(1) if w is not None else 0,
            4 * w.stride(0) if w is not None else 0, space.data_ptr(), need, None)

    torch.cuda.synchronize()
    want = c.want(softcap=20.0, slopes=slopes.cpu(), weights=w)
    assert attend() == 0
    torch.cuda.synchronize()
    R.check(out, *want[:2])
    R.check(w, *want[2:])
    assert attend(sc=None, w=None) == 0
    torch.cuda.synchronize()
    R.check(out, *c.want())
    for kw, text in ((dict(need=need - 1), b"workspace"), (dict(scale=float("inf")), b"scale"),
                     (dict(sc=_lib.Scores(-1.0, 0, None, None, None)), b"softcap"),
                     (dict(sc=_lib.Scores(float("inf"), 0, None, None, None)), b"softcap"),
                     (dict(sc=_lib.Scores(1.0, -1, None, None, None)), b"window"),
                     (dict(sc=_lib.Scores(1.0, 0, 2, None, None)), b"aligned")):
        assert attend(**kw) == -1 and text in L.adaptq_last_error(), (kw, L.adaptq_last_error())
    torch.cuda.synchronize()
    L.adaptq_paged_destroy(h)
