"""Rotations and appends of as many tokens as a call takes: more than the blocks of one launch,
and counts at the end of an int."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    globals().update(PagedCache=PagedCache, Rotary=Rotary)
    yield
    torch.cuda.empty_cache()  # the large tensors go back to the device


def test_rotary_of_more_blocks_than_a_launch():
    """A token of 513 heads is a block of its own, and there are 2^24 + 5 of them (34 GB)."""
    tokens, heads = 2 ** 24 + 5, 513
    x = torch.empty(tokens, heads, 2, dtype=torch.bfloat16, device="cuda")
    x[...] = 1.0
    at = [0, 1, 2 ** 24 - 2, 2 ** 24 - 1, 2 ** 24, tokens - 1]
    x[at] = torch.randn(len(at), heads, 2, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    want = R.rotate(x[at], pos[at], 2)
    Rotary(2)(pos, x, inplace=True)
    R.check(x[at], *want)
    # every token was turned: what (1, 1) becomes has the length of (1, 1) in bf16, and a few
    # thousand of them are checked in full
    some = torch.arange(7, tokens, 4099)
    some = some[(some[:, None] != torch.tensor(at)).all(1)]
    one = torch.ones(len(some), 1, 2, dtype=torch.bfloat16)
    R.check(x[some.cuda(), 100:101], *R.rotate(one, some.int(), 2))


def test_rotary_at_the_end_of_an_int():
    """2^31 - 2 tokens of one pair (8.6 GB): rounded up to whole blocks they pass an int."""
    batch, tokens = 42966, 49981
    assert batch * tokens == 2 ** 31 - 2
    x = torch.empty(batch, tokens, 1, 2, dtype=torch.float16, device="cuda")
    x[..., 0], x[..., 1] = 1.0, 0.5
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    Rotary(2)(pos, x, inplace=True)
    for b in (0, 1, batch // 2, batch - 1):
        one = torch.tensor([1.0, 0.5], dtype=torch.float16).expand(tokens, 1, 2)
        R.check(x[b], *R.rotate(one, pos, 2))
    assert torch.equal(x[1:], x[:1].expand_as(x[1:]))


def test_append_of_more_blocks_than_a_launch():
    """2^24 + 60 tokens of 65 heads, a block each, one row for all of them: the first sequence
    has room for 16, the last for its 10."""
    tokens, heads, dim = 2 ** 24 + 60, 65, 64
    cache = PagedCache.allocate(3, heads, 16, dim, dtype=torch.float32, rotary=Rotary(dim))
    cache.k_pages[...], cache.v_pages[...] = 5.0, 5.0
    row = torch.randn(1, heads, 2 * dim + 1, generator=torch.Generator().manual_seed(1)).cuda()
    k, v = (row[:, :, at:at + dim].expand(tokens, heads, dim) for at in (1, dim + 1))
    table = torch.tensor([[0], [2]], dtype=torch.int32).cuda()
    lengths = torch.tensor([3, 4], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 2 ** 24 + 50, tokens], dtype=torch.int32).cuda()
    cache.append(k, v, table, lengths, offsets)
    for page, first, n in ((0, 3, 13), (2, 4, 10)):
        at = torch.arange(first, first + n)
        want, tol = R.rotate(k[:n].cpu(), at, dim)
        R.check(cache.k_pages[page, :, at.cuda()].transpose(0, 1), want, tol)
        assert torch.equal(cache.v_pages[page, :, at.cuda()].transpose(0, 1), v[:n])
        cache.k_pages[page, :, at.cuda()] = 5.0
        cache.v_pages[page, :, at.cuda()] = 5.0
    assert (cache.k_pages == 5.0).all() and (cache.v_pages == 5.0).all()


def test_append_at_the_end_of_an_int():
    """2^31 - 1 tokens, several a block, all but the last left out."""
    tokens, heads, dim = 2 ** 31 - 1, 1, 8
    cache = PagedCache.allocate(1, heads, 16, dim, dtype=torch.bfloat16)
    cache.k_pages[...], cache.v_pages[...] = 5.0, 5.0
    row = torch.randn(2, 1, heads, dim, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    table = torch.tensor([[-1], [0]], dtype=torch.int32).cuda()
    lengths = torch.tensor([0, 15], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, tokens - 1, tokens], dtype=torch.int32).cuda()
    cache.append(row[0].expand(tokens, heads, dim), row[1].expand(tokens, heads, dim), table,
                 lengths, offsets)
    assert torch.equal(cache.k_pages[0, :, 15], row[0, 0]) and (cache.k_pages[0, :, :15] == 5).all()
    assert torch.equal(cache.v_pages[0, :, 15], row[1, 0]) and (cache.v_pages[0, :, :15] == 5).all()


@pytest.mark.parametrize("n", [2 ** 31 - 34, 2 ** 31 - 33, 2 ** 31 - 32, 2 ** 31 - 5, 2 ** 31 - 1])
def test_step_is_append_then_attend_at_the_last_positions(n):
    """A token at 2^31 - 33 is a sequence's last, for an append as for a step."""
    a, b = (PagedCache.allocate(2, 1, 65536, 8, dtype=torch.float32, rotary=Rotary(8))
            for _ in range(2))
    g = torch.Generator().manual_seed(0)
    for p, r in ((a.k_pages, b.k_pages), (a.v_pages, b.v_pages)):
        p.copy_(torch.randn(p.shape, generator=g))
        r.copy_(p)
    before = a.v_pages.clone()
    table = torch.tensor([[0] * 32768, [1] * 32768], dtype=torch.int32).cuda()
    lengths = torch.tensor([n, 70000], dtype=torch.int32).cuda()
    q, k, v = (torch.randn(2, h, 8, generator=g).cuda() for h in (2, 1, 1))
    got = a.step(q, k, v, table, lengths, window=100)
    b.append(k, v, table, lengths)
    assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)
    assert torch.equal(a.v_pages[0], before[0]) == (n > 2 ** 31 - 33)
    if n < 2 ** 31 - 1:
        assert torch.equal(got, b.attend(q, table, lengths + 1, window=100))
