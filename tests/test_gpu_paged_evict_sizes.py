"""Eviction where `keep` comes near the end of an int: no count of tokens passes it (takes 26 GB)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    globals().update(PagedCache=PagedCache)
    yield
    torch.cuda.empty_cache()


def cache_of(page_size):
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(3, 1, page_size, 8, generator=g).cuda() for _ in range(2))
    return PagedCache(k, v)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("keep", [2 ** 31 - 1, 2 ** 31 - 1000, 2 ** 31 - 1025])
def test_more_than_a_sequence_holds(into, keep):
    """All of its tokens stay: copied whole, or where they are."""
    c = cache_of(65536)
    k0, v0 = c.k_pages.clone(), c.v_pages.clone()
    table = torch.tensor([[1]], dtype=torch.int32).cuda()
    lengths = torch.tensor([100], dtype=torch.int32).cuda()
    w = torch.rand(1, 1, 65536, device="cuda")
    before = w.clone()
    to = torch.full((1, 32768), -1, dtype=torch.int32).cuda()
    to[0, 0] = 2
    kept = c.evict(w, table, lengths, keep, recent=keep, into=to if into else None)
    assert kept.shape == (1, 1, keep) and torch.equal(w, before)
    assert torch.equal(kept[0, 0, :100].cpu(), torch.arange(100, dtype=torch.int32))
    assert (kept[0, 0, 100:] == -1).all()
    if into:
        k0[2, :, :100], v0[2, :, :100] = k0[1, :, :100], v0[1, :, :100]
    assert torch.equal(c.k_pages, k0) and torch.equal(c.v_pages, v0)


def test_nearly_all_of_the_longest_sequence():
    """2^31 - 40 tokens of which 2^31 - 100 stay, in place: the last pages alone are there."""
    n, keep = 2 ** 31 - 40, 2 ** 31 - 100
    c = cache_of(65536)
    v0 = c.v_pages.clone()
    table = torch.full((1, 32768), -1, dtype=torch.int32)
    table[0, -1] = 2
    w = torch.zeros(1, 1, 2 ** 31, device="cuda")
    w[0, 0, 70] = 1.0
    w[0, 0, n - 1] = 2.0
    kept = c.evict(w, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), keep, recent=keep)
    assert kept[0, 0, 0] == 60 and kept[0, 0, -1] == n - 1
    assert w[0, 0, 10] == 1.0 and w[0, 0, keep - 1] == 2.0 and (w[0, 0, keep:] == 0).all()
    assert int((w != 0).sum()) == 2
    end = keep - 32767 * 65536  # places of the last page that are kept
    assert torch.equal(c.v_pages[2, :, :end], v0[2, :, 60:end + 60])
    assert torch.equal(c.v_pages[2, :, end:], v0[2, :, end:])
    assert torch.equal(c.v_pages[:2], v0[:2])
