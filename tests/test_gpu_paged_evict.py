"""Eviction by accumulated weight (PagedCache.evict): what stays is what sorting by (largest
weight, lowest index) leaves, and rows and weights move bit for bit, in place and into other
pages; a serving loop that attends, evicts and goes on."""
import math

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


def choose(w, n, keep, recent):
    """Indexes that stay of a list of weights, by the rule itself."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    best = sorted(range(old), key=lambda t: (-w[t], t))[:keep - recent]
    return sorted(best) + list(range(old, n))


class Case:
    def __init__(self, lengths, heads, dim, ps, dtype, keep, *, seed=0, kind="random", room=0):
        self.p = p = S.Pool(lengths, heads, dim, ps, dtype, seed=seed,
                            spare=3 + len(lengths) * -(-keep // ps))
        self.cache = PagedCache(p.k_pages, p.v_pages)
        tokens = p.table.shape[1] * ps
        w = torch.rand(len(lengths), heads, tokens + room, generator=p.g)
        if kind == "ties":
            w = (w * 4).floor() / 4
        elif kind == "equal":
            w.fill_(0.25)
        elif kind == "zeros":
            w = torch.where(w < 0.6, 0.0, w)
            w = torch.where((w == 0) & (torch.rand(w.shape, generator=p.g) < 0.5), -0.0, w)
        elif kind == "signs":
            w = (w - 0.5) * torch.exp(20 * torch.randn(w.shape, generator=p.g))
        elif kind == "wide":
            w = torch.exp(-80 * w)  # down to denormal numbers
        self.w = w
        need = -(-keep // ps)
        self.into = torch.tensor([p.free[i * need:(i + 1) * need] for i in range(len(lengths))],
                                 dtype=torch.int32).cuda()

    def check(self, keep, recent=0, into=False, weights=None):
        p = self.p
        w = self.w.cuda() if weights is None else weights
        k0, v0 = p.k_pages.cpu(), p.v_pages.cpu()
        kept = self.cache.evict(w, p.table, p.lengths, keep, recent=recent,
                                into=self.into if into else None)
        kept, got = kept.cpu(), w.cpu()
        k1, v1 = p.k_pages.cpu(), p.v_pages.cpu()
        want_k, want_v = k0.clone(), v0.clone()
        table = p.table_host.long()
        to = self.into.cpu().long() if into else table
        for i, n in enumerate(p.held):
            for h in range(p.heads):
                c = choose(self.w[i, h].tolist(), n, keep, recent)
                assert kept[i, h, :len(c)].tolist() == c, (i, h)
                assert (kept[i, h, len(c):] == -1).all()
                x = self.w[i, h].clone()
                if n > keep:
                    x[:keep] = self.w[i, h, c]
                    x[keep:n] = 0
                assert torch.equal(got[i, h], x), (i, h)
                s, d = torch.tensor(c, dtype=torch.int64), torch.arange(len(c))
                if n > keep or into:
                    for want, old in ((want_k, k0), (want_v, v0)):
                        want[to[i, d // p.ps], h, d % p.ps] = old[table[i, s // p.ps], h, s % p.ps]
        for a, b in ((k1, want_k), (v1, want_v)):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        return kept


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("dim", [8, 40, 64, 96, 128, 256])
def test_sizes(dtype, into, dim):
    Case([0, 1, 29, 30, 31, 64, 200, 333], 2, dim, 16, dtype, 30, seed=dim).check(30, 7, into)


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "zeros", "signs", "wide"])
@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (100, 0), (100, 99), (100, 100), (255, 30)])
def test_weights(kind, into, keep, recent):
    Case([1000, 257, 100, 101, 256], 3, 64, 32, torch.bfloat16, keep, kind=kind).check(
        keep, recent, into)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("n,keep,recent", [(5000, 2000, 100), (33000, 32000, 0), (40000, 10, 3),
                                           (70000, 35000, 1000)])
def test_long(into, n, keep, recent):
    """More than 32,768 tokens too."""
    Case([n, 1024, 1025], 1, 16, 64, torch.float16, keep, kind="ties").check(keep, recent, into)


@pytest.mark.parametrize("into", [False, True])
def test_infinite_weights(into):
    c = Case([300], 1, 64, 16, torch.float32, 40)
    c.w[0, 0, 17], c.w[0, 0, 200], c.w[0, 0, 30] = float("inf"), float("inf"), -float("inf")
    c.check(40, 0, into)
    c = Case([300], 1, 64, 16, torch.float32, 40)
    c.w[0, 0, 100] = float("nan")  # counts as larger than all
    kept = c.cache.evict(c.w.cuda(), c.p.table, c.p.lengths, 5)
    assert 100 in kept[0, 0].tolist()


def test_strided_weights():
    c = Case([100, 64, 20], 2, 64, 16, torch.bfloat16, 30)
    room = torch.full((4, 4, c.w.shape[2] + 9), 5.0, device="cuda")
    w = room[1:, 1:3, 4:4 + c.w.shape[2]]
    w.copy_(c.w)
    c.check(30, 3, weights=w)
    w.fill_(5.0)
    assert (room == 5.0).all()


@pytest.mark.parametrize("into", [False, True])
def test_pages_that_are_not_there(into):
    """Rows without a page, or without one to go to, are not moved; nothing else changes."""
    c = Case([200], 1, 64, 16, torch.bfloat16, 64)
    p = c.p
    p.table_host[0, 9] = -1
    p.table.copy_(p.table_host[:, :p.table.shape[1]])
    c.into[0, 1] = 10 ** 9
    k0 = p.k_pages.cpu()
    kept = c.cache.evict(c.w.cuda(), p.table, p.lengths, 64, into=c.into if into else None)[0, 0].tolist()
    want = k0.clone()
    to = c.into[0].tolist() if into else p.table_host[0].tolist()
    for j, s in enumerate(kept):
        a, b = int(p.table_host[0, s // 16]), to[j // 16]
        if 0 <= a < p.pages and 0 <= b < p.pages:
            want[b, 0, j % 16] = k0[a, 0, s % 16]
    assert torch.equal(p.k_pages.cpu().nan_to_num(7.0), want.nan_to_num(7.0))


def test_offsets_beyond_32_bits():
    pages, heads, ps, dim = 70000, 4, 64, 128
    k, v = (torch.zeros(pages, heads, ps, dim, dtype=torch.bfloat16, device="cuda")
            for _ in range(2))
    k[69999], v[69998] = 3.0, 5.0
    cache = PagedCache(k, v)
    table = torch.tensor([[69999, 1, 69998]], dtype=torch.int32).cuda()
    w = torch.zeros(1, heads, 192, device="cuda")
    w[:, :, 128:160] = 1.0
    kept = cache.evict(w, table, torch.tensor([180], dtype=torch.int32).cuda(), 32)
    assert (kept == torch.arange(128, 160, dtype=torch.int32).cuda()).all()
    assert (v[69999, :, :32] == 5.0).all() and (k[69999, :, :32] == 0.0).all()
    assert (k[69999, :, 32:] == 3.0).all()


def test_captured_and_replayed():
    c = Case([500, 300], 2, 64, 16, torch.bfloat16, 100)
    p = c.p
    w = c.w.cuda()
    run = lambda: c.cache.evict(w, p.table, p.lengths, 100, recent=10, into=c.into)  # noqa: E731
    run()
    w.copy_(c.w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run()
    for i in range(4):
        fresh = torch.rand(c.w.shape, generator=p.g)
        w.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        got, moved = kept.clone(), w.clone()
        w.copy_(fresh)
        assert torch.equal(run(), got) and torch.equal(w, moved)
        for b, n in enumerate(p.held):
            assert got[b, 1].tolist() == choose(fresh[b, 1].tolist(), n, 100, 10)


@pytest.mark.parametrize("dtype", DTYPES)
def test_serving_loop(dtype):
    """Prompts, steps whose weights add up, eviction when a budget is reached, and on: every
    output against the 64-bit attention over the tokens that are still there."""
    heads, group, dim, ps, budget = 2, 3, 64, 16, 48
    g = torch.Generator().manual_seed(3)
    p = S.Pool([0, 0, 0], heads, dim, ps, dtype, extra=96)
    cache = PagedCache(p.k_pages, p.v_pages)
    prompt = [40, 7, 60]

    def normal(*shape):
        return torch.randn(shape, generator=g).to(dtype)

    k, v, q = normal(sum(prompt), heads, dim), normal(sum(prompt), heads, dim), \
        normal(sum(prompt), heads * group, dim)
    offsets = S.spans(prompt)
    lengths = torch.zeros(3, dtype=torch.int32).cuda()
    cache.append(k.cuda(), v.cuda(), p.table, lengths, offsets)
    lengths += offsets[1:] - offsets[:-1]
    out = cache.attend(q.cuda(), p.table, lengths, offsets, softcap=30.0)
    at = [0, 40, 47, 107]
    held = []  # per sequence and head: keys and values that are there
    for i, n in enumerate(prompt):
        rows = slice(at[i], at[i + 1])
        pos = torch.arange(n)
        seen = S.sees(n, pos, torch.zeros(n), torch.zeros(n), None)
        o, t, _, _ = S.attend(q[rows].double(), k[rows].transpose(0, 1), v[rows].transpose(0, 1),
                              seen, pos, 1 / math.sqrt(dim), dtype, softcap=30.0,
                              rough=dtype != torch.float32)
        R.check(out[at[i]:at[i + 1]], o, t)
        held.append([[k[rows][:, h], v[rows][:, h]] for h in range(heads)])
    weights = torch.zeros(3, heads, p.table.shape[1] * ps, device="cuda")
    evicted = False
    for step in range(40):
        k, v, q = normal(3, heads, dim), normal(3, heads, dim), normal(3, heads * group, dim)
        out = cache.step(q.cuda(), k.cuda(), v.cuda(), p.table, lengths, softcap=30.0,
                         weights=weights)
        lengths += 1
        for i in range(3):
            for h in range(heads):
                for j, x in enumerate((k, v)):
                    held[i][h][j] = torch.cat((held[i][h][j], x[i, h][None]))
                kk, vv = held[i][h]
                n = kk.shape[0]
                seen = torch.ones(1, n, dtype=torch.bool)
                o, t, _, _ = S.attend(q[i:i + 1, h * group:(h + 1) * group].double(), kk[None],
                                      vv[None], seen, torch.tensor([n - 1]), 1 / math.sqrt(dim),
                                      dtype, softcap=30.0)
                R.check(out[i:i + 1, h * group:(h + 1) * group], o, t, f"step {step}")
        if step % 8 == 7:
            kept = cache.evict(weights, p.table, lengths, budget, recent=8).cpu()
            lengths.clamp_(max=budget)
            for i in range(3):
                for h in range(heads):
                    c = kept[i, h][kept[i, h] >= 0].long()
                    n = held[i][h][0].shape[0]
                    assert len(c) == min(n, budget)
                    evicted = evicted or n > budget
                    held[i][h] = [x[c] for x in held[i][h]]
    assert evicted


def test_refusals():
    c = Case([50, 30], 2, 64, 16, torch.bfloat16, 20)
    w, t, n = c.w.cuda(), c.p.table, c.p.lengths
    for kw in (dict(keep=0), dict(keep=-1), dict(keep=10, recent=11), dict(keep=10, recent=-1),
               dict(keep=20, into=c.into[:, :1]), dict(keep=20, into=c.into.long()),
               dict(keep=20, into=c.into.cpu()), dict(keep=20, into=c.into[:1])):
        with pytest.raises(ValueError):
            c.cache.evict(w, t, n, **kw)
    for bad in (w[:1], w.half(), w.cpu(), w[:, :, 1:]):
        with pytest.raises(ValueError):
            c.cache.evict(bad, t, n, 10)
    pages = c.p.v_pages.flatten().view(torch.float32)[:w.numel()].view(w.shape)
    with pytest.raises(RuntimeError, match="overlap"):
        c.cache.evict(pages, t, n, 10)
    rotates = PagedCache(c.p.k_pages, c.p.v_pages, rotary=Rotary(64))
    with pytest.raises(ValueError):
        rotates.evict(w, t, n, 10)
