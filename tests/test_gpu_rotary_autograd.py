"""What torch sees of Rotary and PagedCache on the GPU: tangents, tensors written in place,
traced calls."""
import pytest
import torch
from torch.autograd import forward_ad

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Rotary(torch_dev):
    from adaptq_amd.rotary import Rotary
    return Rotary


def _rows(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved,rot,dim", [(False, 64, 64), (True, 32, 80)])
def test_tangents(Rotary, dtype, interleaved, rot, dim):
    """The tangent of the outputs is the rotated tangent, on strided views too."""
    rotary = Rotary(rot, interleaved=interleaved, scaling="yarn", factor=4.0, context=2048)
    kw = dict(scaling="yarn", factor=4.0, context=2048)
    pos = torch.arange(70, 75, dtype=torch.int32).cuda()
    base, tangent = _rows((2, 5, 7, dim), dtype), _rows((2, 5, 7, dim), dtype, 1)
    p = pos.expand(2, 5)
    with forward_ad.dual_level():
        q = forward_ad.make_dual(base[:, :, :4], tangent[:, :, :4])
        k = forward_ad.make_dual(base[:, :, 4:6], tangent[:, :, 4:6])
        for y, x, t in zip(rotary(pos, q, k), (base[:, :, :4], base[:, :, 4:6]),
                           (tangent[:, :, :4], tangent[:, :, 4:6])):
            y, d = forward_ad.unpack_dual(y)
            R.check(y, *R.rotate(x, p, rot, interleaved, **kw))
            R.check(d, *R.rotate(t, p, rot, interleaved, **kw))
        # the tangent of a gradient, on leaves that need one
        x = base[:, :, :4].detach().requires_grad_()
        (dx,) = torch.autograd.grad(rotary(pos, x), (x,), q)
        y, d = forward_ad.unpack_dual(dx)
        R.check(d, *R.rotate(tangent[:, :, :4], p, rot, interleaved, backward=True, **kw))


def test_written_in_place(Rotary):
    from adaptq_amd.paged import PagedCache
    rotary, pos = Rotary(64), torch.arange(4, dtype=torch.int32).cuda()
    q, k = _rows((4, 2, 64), torch.float32), _rows((4, 1, 64), torch.float32, 1)
    w = torch.ones(64, device="cuda", requires_grad=True)
    for x, call in ((q, lambda: rotary(pos, q, inplace=True)),
                    (k, lambda: rotary(pos, q, k, inplace=True))):
        z = (w * x).sum()
        with torch.no_grad():
            call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    cache = PagedCache.allocate(4, 2, 16, 64, dtype=torch.float32)
    table = torch.arange(4, dtype=torch.int32).cuda()[:, None]
    lengths = torch.zeros(4, dtype=torch.int32).cuda()
    z = (w * cache.v_pages).sum()
    cache.step(q, q, q, table, lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_traced_calls_are_refused(Rotary):
    from torch.fx.experimental.proxy_tensor import make_fx
    rotary, pos, q = Rotary(64), torch.arange(4, dtype=torch.int32).cuda(), \
        _rows((4, 2, 64), torch.float32)
    for trace in (lambda f: make_fx(f)(q), lambda f: torch.jit.trace(f, (q,), check_trace=False)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace(lambda x: rotary(pos, x) + 1)
    R.check(rotary(pos, q), *R.rotate(q, pos, 64))
