"""One PagedCache used on several streams that the caller has not ordered."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    globals().update(PagedCache=PagedCache)


def _cache(n, tokens, heads, dim, page=64):
    g = torch.Generator().manual_seed(n)
    width = -(-(tokens + 40) // page)
    k, v = (torch.randn(n * width, heads, page, dim, generator=g).bfloat16().cuda()
            for _ in range(2))
    table = torch.arange(n * width, dtype=torch.int32).view(n, width).cuda()
    return (PagedCache(k, v), table, torch.full((n,), tokens, dtype=torch.int32).cuda(),
            lambda *s: torch.randn(*s, generator=g).bfloat16().cuda())


def test_attends_on_two_streams():
    """Calls that would run over each other's workspace: each gives its own result, and so does
    every call after them."""
    cache, table, lengths, normal = _cache(2, 20000, 2, 64)
    qs = [normal(2, h, 64) for h in (2, 32, 6)]
    want = [cache.attend(q, table, lengths, window=w) for q, w in zip(qs, (None, 9000, 15000))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cache.attend(qs[i % 3], table, lengths, window=(None, 9000, 15000)[i % 3]))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 3]), i
    for q, w, y in zip(qs, (None, 9000, 15000), want):
        assert torch.equal(cache.attend(q, table, lengths, window=w), y)
    # and the results are right
    k, v = (p.view(2, -1, 2, 64, 64).transpose(1, 2).reshape(2, 2, -1, 64)[:, :, :20000].cpu()
            for p in (cache.k_pages, cache.v_pages))
    for i in range(2):
        o, t = R.attend(qs[0][i].cpu().double().view(2, 1, 64), k[i], v[i], 1 / math.sqrt(64),
                        torch.bfloat16)
        R.check(want[0][i], o.view(2, 64), t.view(2, 64))


def test_steps_alternate_between_streams():
    """Rows that one stream appends are there for the next one's attention."""
    a, table, lengths, normal = _cache(3, 5000, 2, 64)
    b = PagedCache(a.k_pages.clone(), a.v_pages.clone())
    streams = [torch.cuda.Stream() for _ in range(3)] + [torch.cuda.default_stream()]
    calls = [(normal(3, 8, 64), normal(3, 2, 64), normal(3, 2, 64), lengths + i) for i in range(24)]
    torch.cuda.synchronize()
    got = []
    for i, (q, k, v, n) in enumerate(calls):
        with torch.cuda.stream(streams[i % 4]):
            if i % 3 == 2:
                a.append(k, v, table, n)
            else:
                got.append(a.step(q, k, v, table, n))
    torch.cuda.synchronize()
    want = []
    for i, (q, k, v, n) in enumerate(calls):
        if i % 3 == 2:
            b.append(k, v, table, n)
        else:
            want.append(b.step(q, k, v, table, n))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)


def test_captured_calls_do_not_wait_for_streams_outside():
    """A capture takes nothing from another stream; its replays are ordered by the caller."""
    cache, table, lengths, normal = _cache(1, 3000, 2, 64)
    q = normal(1, 4, 64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        want = cache.attend(q, table, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, table, lengths)
        again = cache.attend(q, table, lengths, window=100)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(cache.attend(q, table, lengths, window=100), again)
        torch.cuda.synchronize()


@pytest.mark.parametrize("heads", [4, 64])
def test_replays_and_calls_share_the_workspace(heads):
    """A captured step replayed, its lengths advancing, with eager attention over other lengths
    between the replays: both sides' values are those of a cache of their own."""
    a, table, lengths, normal = _cache(3, 6000, 2, 64)
    b = PagedCache(a.k_pages.clone(), a.v_pages.clone())
    own, other = lengths.clone(), torch.tensor([6000, 17, 3100], dtype=torch.int32).cuda()
    q, k, v = normal(3, heads, 64), normal(3, 2, 64), normal(3, 2, 64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step(q, k, v, table, own)
        own.add_(1)
    for i in range(5):
        for x in (q, k, v):
            x.copy_(normal(*x.shape))
        graph.replay()
        eager = a.attend(q, table, other)
        want = b.step(q, k, v, table, lengths)
        lengths += 1
        assert torch.equal(out, want) and torch.equal(own, lengths), i
        assert torch.equal(eager, b.attend(q, table, other)), i
        assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)
        torch.cuda.synchronize()


@pytest.mark.parametrize("captured_last", [True, False])
def test_calls_beside_a_capture_stay_outside_it(captured_last):
    """An eager call while the stream of the last call (or another) is being captured runs at
    once: waiting for a captured stream would make the call a part of the graph."""
    cache, table, lengths, normal = _cache(1, 3000, 2, 64)
    q, out = normal(1, 4, 64), torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    want = cache.attend(q, table, lengths)
    x = torch.zeros(1, device="cuda")
    stream, other, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    if captured_last:
        with torch.cuda.stream(stream):
            cache.attend(q, table, lengths)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        x.add_(1)
        with torch.cuda.stream(other):
            cache.attend(q, table, lengths, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert x.item() == i + 1 and not out.any()
