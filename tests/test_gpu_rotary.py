"""Rotary positions (adaptq_rotary_*, adaptq_amd.rotary) against the formula in 64 bits:
types, layouts, partial rotation, scalings, far and negative positions, strides, in place,
gradients, streams, graphs; and what a call refuses."""
import ctypes as C

import pytest
import torch

import paged_ref as R
from adaptq_amd import _lib

pytestmark = pytest.mark.gpu
L = _lib.lib
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def Rotary(torch_dev):
    from adaptq_amd.rotary import Rotary
    return Rotary


def _rows(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def _positions(n, first=0):
    return torch.arange(first, first + n, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot,tokens,hq,hk", [
    (64, 64, 1, 14, 14), (128, 128, 7, 32, 8), (128, 64, 33, 5, 1), (80, 80, 9, 3, 3),
    (80, 40, 9, 6, 2), (96, 24, 17, 4, 1), (256, 256, 3, 2, 1), (10, 6, 5, 3, 2), (7, 2, 4, 2, 1),
    (2, 2, 300, 1, 1), (1024, 1024, 3, 2, 2), (1000, 12, 2, 3, 1), (64, 64, 4099, 2, 1),
    (72, 36, 2049, 8, 1),
])
def test_formula(Rotary, dtype, interleaved, dim, rot, tokens, hq, hk):
    q, k = _rows((tokens, hq, dim), dtype, 1), _rows((tokens, hk, dim), dtype, 2)
    pos = _positions(tokens, 11)
    q0, k0 = q.clone(), k.clone()
    got = Rotary(rot, interleaved=interleaved)(pos, q, k)
    for x, y in zip((q, k), got):
        assert y.dtype == dtype and y.shape == x.shape
        R.check(y, *R.rotate(x, pos, rot, interleaved))
    assert torch.equal(q, q0) and torch.equal(k, k0)


@pytest.mark.parametrize("first", [0, 1, 4095, 131071, 1000003, 2 ** 31 - 9, -1, -2 ** 31, -77777])
def test_far_positions(Rotary, first):
    """fp32 rows far from 0: the angle stays exact (its whole turns drop out)."""
    q, pos = _rows((8, 3, 128), torch.float32), _positions(8, first)
    for kw in ({}, {"base": 1.5}, {"base": 5e5, "scaling": "linear", "factor": 32.0}):
        # fp64 holds position * angle to 2^31 * 2^-53 = 2^-22 radians at the farthest: as much
        # again as the fp32 rotation's own error is allowed beside it
        want, tol = R.rotate(q, pos, 128, **kw)
        far = abs(first) * 2.0 ** -52 * 4
        R.check(Rotary(128, **kw)(pos, q), want, tol + far * q.cpu().double().abs().amax(-1, True) * 2)


@pytest.mark.parametrize("kw", [
    dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0, base=500000.0),
    dict(scaling="yarn", factor=16.0, context=4096), dict(scaling="yarn", factor=1.0, context=64),
    dict(scaling="yarn", factor=4.0, context=2048, slow=2.0, fast=20.0, amplitude=1.25),
    dict(scaling="bands", factor=8.0, context=8192, base=500000.0),
    dict(scaling="bands", factor=2.0, context=2, slow=0.5, fast=3.0),
    dict(amplitude=0.75),
])
@pytest.mark.parametrize("rot", [128, 20])
def test_scalings(Rotary, kw, rot):
    q, pos = _rows((50, 2, 128), torch.float32), _positions(50, 30000)
    R.check(Rotary(rot, **kw)(pos, q), *R.rotate(q, pos, rot, **kw))


def test_batches_share_or_have_positions(Rotary):
    q, k = _rows((3, 5, 4, 64), torch.bfloat16), _rows((3, 5, 2, 64), torch.bfloat16, 1)
    rotary = Rotary(64)
    one = _positions(5, 9)
    each = torch.randint(0, 9999, (3, 5), dtype=torch.int32).cuda()
    for pos, p in ((one, one.expand(3, 5)), (one[None], one.expand(3, 5)), (each, each),
                   (each.t().contiguous().t(), each)):
        for x, y in zip((q, k), rotary(pos, q, k)):
            R.check(y, *R.rotate(x, p, 64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inplace", [False, True])
def test_strided_views(Rotary, dtype, inplace):
    """Views of one projection, heads-first rows, rows that start off alignment, and a
    stride-0 batch read; the memory around the outputs stays as it was."""
    b, t, hq, hk, d = 2, 6, 4, 2, 64
    rotary, pos = Rotary(32), _positions(6, 100)
    for pad in (0, 1, 2):
        fused = _rows((b, t, hq + 2 * hk + 1, d + pad), dtype)
        before = fused.clone()
        q, k = fused[:, :, :hq, pad:], fused[:, :, hq:hq + hk, pad:]
        want = [R.rotate(x, pos.expand(b, t), 32) for x in (q, k)]
        got = rotary(pos, q, k, inplace=inplace)
        for y, w in zip(got, want):
            R.check(y, *w)
        if inplace:
            assert got[0] is q and got[1] is k
            before[:, :, :hq, pad:], before[:, :, hq:hq + hk, pad:] = q, k
        assert torch.equal(fused, before)
    heads_first = _rows((b, hq, t, d), dtype).transpose(1, 2)
    y = rotary(pos, heads_first, inplace=inplace)
    if not inplace:
        R.check(y, *R.rotate(heads_first, pos.expand(b, t), 32))
        wide = _rows((1, t, hq, d), dtype).expand(b, t, hq, d)
        R.check(rotary(pos, wide), *R.rotate(wide, pos.expand(b, t), 32))
        turned = _rows((t, d, hq), dtype).transpose(1, 2)  # values of a row not side by side
        R.check(rotary(pos, turned), *R.rotate(turned, pos, 32))


def test_infinities_and_nan_stay_in_their_pair(Rotary):
    q = _rows((4, 2, 64), torch.float32)
    bad = q.clone()
    bad[1, 0, 3], bad[2, 1, 40] = float("nan"), float("inf")
    pos = _positions(4, 5)
    a, b = Rotary(64)(pos, q), Rotary(64)(pos, bad)
    touched = torch.zeros_like(q, dtype=torch.bool)
    touched[1, 0, [3, 35]] = touched[2, 1, [8, 40]] = True
    assert torch.equal(a[~touched], b[~touched])
    assert not torch.isfinite(b[touched]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved,rot,dim", [(False, 64, 64), (True, 32, 80)])
def test_gradients(Rotary, dtype, interleaved, rot, dim):
    kw = dict(scaling="yarn", factor=4.0, context=2048)
    rotary = Rotary(rot, interleaved=interleaved, **kw)
    pos = _positions(5, 70)
    base = _rows((2, 5, 7, dim), dtype)  # leaves are views of one tensor
    q, k = base[:, :, :4].detach().requires_grad_(), base[:, :, 4:6].detach().requires_grad_()
    yq, yk = rotary(pos, q, k)
    gq, gk = _rows(yq.shape, dtype, 5), _rows(yk.shape, dtype, 6)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    p = pos.expand(2, 5)
    for d, g in ((dq, gq), (dk, gk)):
        R.check(d, *R.rotate(g, p, rot, interleaved, backward=True, **kw))
    # one of the two, an expanded gradient, and inputs that need none
    yq, yk = rotary(pos, q, k.detach())
    (dq,) = torch.autograd.grad(yq.sum(), (q,))
    one = torch.ones_like(gq)
    R.check(dq, *R.rotate(one, p, rot, interleaved, backward=True, **kw))
    assert not yk.requires_grad
    y = rotary(pos, k)
    (dk,) = torch.autograd.grad(y, (k,), gk)
    R.check(dk, *R.rotate(gk, p, rot, interleaved, backward=True, **kw))


def test_gradient_against_differences(Rotary):
    """The rotation is linear, so a difference of any width is its derivative: (y(x + h w) -
    y(x - h w)) / 2h . g = w . grad.  With h = 1 the only errors are the fp32 roundings,
    2^-20 of the values' size a term (paged_ref.rotate), added over the terms."""
    rotary, pos = Rotary(48, interleaved=True, amplitude=1.5), _positions(9, 1000)
    x, w, g = (_rows((9, 3, 64), torch.float32, i) for i in range(3))
    x.requires_grad_()
    (dx,) = torch.autograd.grad(rotary(pos, x), (x,), g)
    with torch.no_grad():
        diff = (rotary(pos, x + w).double() - rotary(pos, x - w).double()) / 2
    size = (w.double().abs() + x.detach().double().abs()).sum() * g.double().abs().max() * 4
    assert abs((diff * g.double()).sum() - (w.double() * dx.double()).sum()) <= 2.0 ** -20 * size


def test_second_gradient(Rotary):
    rotary, pos = Rotary(16), _positions(3, 2)
    x = _rows((3, 2, 16), torch.float32).requires_grad_()
    g = _rows((3, 2, 16), torch.float32, 1).requires_grad_()
    (dx,) = torch.autograd.grad(rotary(pos, x), (x,), g, create_graph=True)
    h = _rows((3, 2, 16), torch.float32, 2)
    (dg,) = torch.autograd.grad(dx, (g,), h)
    R.check(dg, *R.rotate(h, pos, 16))


def test_side_stream_and_graph(Rotary):
    """On another stream, and captured: a replay follows the positions and rows as they are."""
    rotary, q, pos = Rotary(64), _rows((40, 4, 64), torch.float16), _positions(40)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = rotary(pos, q)
    s.synchronize()
    R.check(y, *R.rotate(q, pos, 64))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        y = rotary(pos, q)
    for i in range(3):
        pos.add_(1000 * i + 1)
        q.copy_(_rows((40, 4, 64), torch.float16, i))
        graph.replay()
        torch.cuda.synchronize()
        R.check(y, *R.rotate(q, pos, 64))
        assert torch.equal(y, rotary(pos, q))


def test_offsets_beyond_32_bits(Rotary):
    """Rows more than 2^32 bytes from the first, of one token set and of a batch."""
    tokens, heads, dim = 140000, 128, 128
    q = torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
    assert q.numel() * 2 > 2 ** 32
    last = _rows((3, heads, dim), torch.bfloat16)
    q[-3:] = last
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    rotary = Rotary(64, interleaved=True)
    want = R.rotate(last, pos[-3:], 64, True)
    y = rotary(pos, q)
    R.check(y[-3:], *want)
    assert not y[:-3].any()
    del y
    rotary(pos.view(20, -1), q.view(20, -1, heads, dim), inplace=True)
    R.check(q[-3:], *want)


def test_captured_backward(Rotary):
    """Forward and gradient in one graph, on leaves that no eager graph holds; replays follow
    the rows, the positions and the outputs' gradient."""
    rotary, pos = Rotary(64), _positions(24, 3)
    q, k = (_rows((24, h, 64), torch.float32, h).requires_grad_() for h in (4, 2))
    gq, gk = torch.empty_like(q), torch.empty_like(k)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        yq, yk = rotary(pos, q, k)
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for i in range(3):
        with torch.no_grad():
            for j, x in enumerate((q, k, gq, gk)):
                x.copy_(_rows(x.shape, torch.float32, 10 * i + j))
            pos.add_(77)
        graph.replay()
        torch.cuda.synchronize()
        for y, x in ((yq, q), (yk, k)):
            R.check(y, *R.rotate(x, pos, 64))
        for d, g in ((dq, gq), (dk, gk)):
            R.check(d, *R.rotate(g, pos, 64, backward=True))


def test_empty(Rotary):
    rotary = Rotary(64)
    for shape in ((0, 4, 64), (0, 5, 4, 64), (2, 0, 4, 64)):
        q = torch.empty(shape, device="cuda")
        pos = torch.empty(shape[:-2][-1:], dtype=torch.int32, device="cuda")
        assert rotary(pos, q).shape == q.shape


def test_refusals(Rotary):
    rotary = Rotary(64)
    q, k, pos = _rows((4, 2, 64), torch.float32), _rows((4, 1, 64), torch.float32), _positions(4)
    cases = [
        (TypeError, (pos.long(), q)), (TypeError, (pos, q.double())),
        (ValueError, (pos[:3], q)), (ValueError, (pos, q[0])), (ValueError, (pos[None], q)),
        (ValueError, (pos, q, k.half())), (ValueError, (pos, q, k[:3])),
        (ValueError, (pos, q, k[..., :32])), (ValueError, (pos.cpu(), q)),
        (ValueError, (pos, q.cpu())), (ValueError, (pos, q, k[:, :0])),
        (RuntimeError, (pos, q[..., :32].contiguous())),
    ]
    for kind, args in cases:
        with pytest.raises(kind):
            rotary(*args)
    with pytest.raises(ValueError):
        rotary(pos, q.requires_grad_(), inplace=True)
    q = q.detach()
    with pytest.raises(RuntimeError, match="overlap"):
        rotary(pos, q[:, :1].expand(4, 2, 64), inplace=True)
    with pytest.raises(RuntimeError, match="overlap"):
        rotary(pos, q, q[:, :1], inplace=True)
    with pytest.raises(ValueError):
        Rotary(2)(pos, q.transpose(1, 2), inplace=True)  # values of a row not side by side
    for kw in (dict(scaling="other"), dict(amplitude=0.0), dict(slow=-1.0), dict(device="cpu")):
        with pytest.raises(ValueError):
            Rotary(64, **kw)


def test_c_refusals(Rotary):
    """The C entry: overlapping outputs, strides and pointers off the element size."""
    r = L.adaptq_rotary_create(64, 0, 10000.0, 0, 1.0, 0, 0.0, 0.0, 0.0)
    assert r, _lib.last_error()
    x = torch.zeros(4096, device="cuda")
    pos = _positions(4)

    def call(n=1, dim=64, io=0, positions=pos.data_ptr(), stride=0, batch=1, tokens=4, **kw):
        base = dict(in_=x.data_ptr(), out=x.data_ptr() + 8192, n_heads=2, in_nb1=256, in_nb2=512,
                    in_nb3=0, out_nb1=256, out_nb2=512, out_nb3=0)
        rows = (_lib.Rows * 2)(_lib.Rows(**{**base, **kw}), _lib.Rows(**base))
        return L.adaptq_rotary_device(r, rows, n, dim, io, positions, stride, batch, tokens, 0, None)

    assert call() == 0, _lib.last_error()
    for kw in (dict(n=0), dict(n=3), dict(dim=62), dict(dim=1025), dict(io=3), dict(io=-1),
               dict(positions=None), dict(stride=3), dict(batch=-1), dict(tokens=-1), dict(in_=None),
               dict(out=None), dict(n_heads=0), dict(in_nb1=258), dict(out_nb2=510),
               dict(in_=x.data_ptr() + 2), dict(out=x.data_ptr() + 256),
               dict(out=x.data_ptr() + 512), dict(out_nb1=128), dict(out_nb2=256),
               dict(out_nb2=0), dict(in_nb2=2 ** 62), dict(n=2),
               dict(batch=2 ** 20, tokens=2 ** 20)):
        assert call(**kw) == -1, kw
        assert _lib.last_error().startswith("adaptq_rotary_device: "), kw
    assert call(tokens=0) == 0 and call(batch=0) == 0
    # side by side in rows of one tensor: nothing is shared
    assert call(in_=x.data_ptr(), in_nb2=1024, out=x.data_ptr() + 512, out_nb2=1024) == 0
    assert call(in_=x.data_ptr(), in_nb2=1024, out=x.data_ptr() + 480, out_nb2=1024) == -1
    torch.cuda.synchronize()
    L.adaptq_rotary_destroy(r)


@pytest.mark.parametrize("dtype", DTYPES)
def test_torch_adapter(Rotary, dtype):
    """AdaptQAttention(rotary=...) is the module without it fed rotated queries and keys: the
    same outputs bit for bit, over the end of the module's positions and after a reset."""
    from adaptq_amd.torch_adapter import AdaptQAttention
    H, D = 3, 64
    rotary = Rotary(32, base=500.0)
    a = AdaptQAttention(D, H, seed=3, rotary=rotary)
    b = AdaptQAttention(D, H, seed=3)
    g = torch.Generator().manual_seed(1)
    for t in [0, *range(4090, 4100), 0, 1, 2]:  # the module holds 4,096 positions at a time
        if t == 0:
            a.reset_cache()
            b.reset_cache()
        a.engine.pos = b.engine.pos = t
        q, k, v = (torch.randn(1, H, D, generator=g).to(dtype).cuda()
                   for _ in range(3))
        q0, k0 = q.clone(), k.clone()
        pos = torch.tensor([t], dtype=torch.int32).cuda()
        rq, rk = rotary(pos, q, k)
        assert torch.equal(a(q, k, v), b(rq, rk, v)), t
        assert torch.equal(q, q0) and torch.equal(k, k0)
    with pytest.raises(ValueError):
        a(q.cpu(), k.cpu(), v.cpu())
    torch.cuda.synchronize()
    graph, y = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            a(q, k, v)
    assert a.engine.pos == 3
