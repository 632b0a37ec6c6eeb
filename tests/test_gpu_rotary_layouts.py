"""Rotation in place, and steps whose output lies among their inputs, on parts of one tensor
whose rows alternate."""
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Rotary(torch_dev):
    from adaptq_amd.rotary import Rotary
    return Rotary


def _rows(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


LAYOUTS = {
    # queries, keys and values of a head side by side, [tokens, heads, 3, dim]
    "per head": ((6, 4, 3, 64), lambda x: (x[:, :, 0], x[:, :, 1])),
    "per head, one token": ((1, 4, 3, 64), lambda x: (x[:, :, 0], x[:, :, 1])),
    "per head, a batch": ((2, 6, 4, 3, 64), lambda x: (x[:, :, :, 0], x[:, :, :, 1])),
    # heads first, queries and keys the halves of a batch's heads
    "heads first": ((2, 6, 5, 64), lambda x: (x[:, :4].transpose(1, 2), x[:, 4:].transpose(1, 2))),
    "every other head": ((2, 5, 8, 64), lambda x: (x[:, :, 0::2], x[:, :, 1::2])),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_in_place(Rotary, dtype, layout):
    shape, parts = LAYOUTS[layout]
    rotary, x = Rotary(32), _rows(shape, dtype)
    before = x.clone()
    q, k = parts(x)
    pos = torch.arange(9, 9 + q.shape[-3], dtype=torch.int32).cuda()
    p = pos.expand(q.shape[:-2])
    want = [R.rotate(y, p, 32) for y in (q, k)]
    got = rotary(pos, q, k, inplace=True)
    assert got[0] is q and got[1] is k
    for y, w, z in zip((q, k), want, parts(before)):
        R.check(y, *w)
        z.copy_(y)
    assert torch.equal(x, before)  # nothing else changed


def test_step_into_its_projection(Rotary):
    """The output in the place of the values' neighbours, one per head."""
    from adaptq_amd.paged import PagedCache
    x = _rows((3, 2, 4, 64), torch.float32)
    q, k, v, out = x.unbind(2)
    caches = [PagedCache(torch.zeros(3, 2, 16, 64).cuda(), torch.zeros(3, 2, 16, 64).cuda(),
                         rotary=Rotary(64)) for _ in range(2)]
    table = torch.arange(3, dtype=torch.int32).cuda()[:, None]
    lengths = torch.tensor([0, 3, 15], dtype=torch.int32).cuda()
    want = caches[0].step(q.clone(), k.clone(), v.clone(), table, lengths)
    before = x.clone()
    assert caches[1].step(q, k, v, table, lengths, out=out) is out
    assert torch.equal(out, want) and torch.equal(x[:, :, :3], before[:, :, :3])
