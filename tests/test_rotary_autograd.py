"""What torch sees of the calls that go to the library by address, on the CPU: the handles'
calls are replaced by the same arithmetic in torch."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad


def _tensor(address, offset_shape_strides):
    """A float32 tensor over memory that another tensor holds."""
    shape, strides = offset_shape_strides
    n = 1 + sum((s - 1) * t for s, t in zip(shape, strides))
    flat = torch.frombuffer((C.c_float * n).from_address(address), dtype=torch.float32)
    return flat.as_strided(shape, strides)


class RotaryHandle:
    """Pairs (i, i + dim/2) by position * 3^-i radians; rows of float32."""
    calls = 0

    def rotate(self, positions, pos_stride, batch, tokens, dim, io, backward, stream, *rows):
        self.calls += 1
        assert io == 0
        at = torch.frombuffer((C.c_int * tokens).from_address(positions), dtype=torch.int32)
        angle = at[:, None].double() * 3.0 ** -torch.arange(dim // 2)
        c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if backward else 1)
        for x, y, heads, x1, x2, x3, y1, y2, y3 in (rows[:9], rows[9:]) if rows[9:] else (rows,):
            shape = batch, tokens, heads, dim
            x = _tensor(x, (shape, (x3 // 4, x2 // 4, x1 // 4, 1))).double()
            a, b = x[..., :dim // 2], x[..., dim // 2:]
            _tensor(y, (shape, (y3 // 4, y2 // 4, y1 // 4, 1))).copy_(
                torch.cat((a * c - b * s, b * c + a * s), -1))


@pytest.fixture
def rotary(monkeypatch):
    from adaptq_amd import rotary as module
    monkeypatch.setattr(module, "stream_of", lambda device: 0)
    r = module.Rotary.__new__(module.Rotary)
    r.dim, r.device, r._handle = 8, torch.device("cpu"), RotaryHandle()
    return r


POS = torch.arange(5, 8, dtype=torch.int32)


def _rows(heads=2, seed=0):
    return torch.randn(3, heads, 8, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("which", [0, 1])
def test_inplace_is_seen_by_graphs_that_saved_the_rows(rotary, mode, which):
    """As torch's own in-place operators: the gradient of w would be of the rotated rows."""
    q, k = _rows(), _rows(1, 1)
    w = torch.randn(8, requires_grad=True)
    z = (w * (q, k)[which]).sum()
    other = (w * 2).sum()
    with mode():
        rotary(POS, q, k, inplace=True)
    other.backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_inplace_of_an_activation(rotary):
    """A view of a projection rotated under no_grad, whose graph a product had saved."""
    x = torch.randn(3, 24, requires_grad=True)
    fused = (x * 1).view(3, 3, 8)
    y = (fused * fused).sum()
    with torch.no_grad():
        rotary(POS, fused[:, :2], inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_rows_of_inference_mode_rotate_in_place(rotary):
    with torch.inference_mode():
        q = _rows()
        want = rotary(POS, q)
        assert torch.equal(rotary(POS, q, inplace=True), want) and torch.equal(q, want)


def test_calls_that_write_nothing_of_the_callers_raise_no_version(rotary):
    q, k = _rows(), _rows(1, 1)
    rotary(POS, q, k)
    assert q._version == 0 and k._version == 0 and POS._version == 0


class PagedHandle:
    def append(self, *a):
        pass

    attend = step = append


@pytest.fixture
def cache(monkeypatch):
    from adaptq_amd import paged as module
    monkeypatch.setattr(module, "stream_of", lambda device: 0)

    # the class checks that its pools are on a GPU: built around that
    c = module.PagedCache.__new__(module.PagedCache)
    c.k_pages, c.v_pages = c._pools = torch.zeros(4, 2, 16, 8), torch.zeros(4, 2, 16, 8)
    c.device, c.dtype, c._size, c._io = torch.device("cpu"), torch.float32, 4, 0
    c.pages, c.heads, c.page_size, c.dim = c.k_pages.shape
    c._handle, c._last_address = PagedHandle(), 0
    return c


def test_pools_and_outputs_are_seen_as_written(cache):
    table, lengths = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q, k, out = _rows(4), _rows(), _rows(4)
    versions = lambda: (cache.k_pages._version, cache.v_pages._version, out._version)  # noqa: E731
    assert versions() == (0, 0, 0)
    cache.append(k, k, table, lengths)
    assert versions() == (1, 1, 0)
    assert cache.attend(q, table, lengths) is not out and versions() == (1, 1, 0)
    assert cache.attend(q, table, lengths, out=out) is out and versions() == (1, 1, 1)
    cache.step(q, k, k, table, lengths)
    assert versions() == (2, 2, 1)
    assert cache.step(q, k, k, table, lengths, out=out) is out and versions() == (3, 3, 2)
    assert q._version == k._version == table._version == lengths._version == 0
    w = torch.ones(8, requires_grad=True)
    z = (w * out).sum()
    cache.attend(q, table, lengths, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def _turned(x, backward=False):
    """The stub's rotation in 64 bits."""
    angle = POS[:, None].double() * 3.0 ** -torch.arange(4)
    c, s = angle.cos()[:, None], angle.sin()[:, None] * (-1 if backward else 1)
    a, b = x.double()[..., :4], x.double()[..., 4:]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _near(got, want):
    # fp64 arithmetic on fp32 rows, rounded once
    assert ((got.double() - want).abs() <= 2.0 ** -23 * want.abs() + 1e-6).all()


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_forward_mode(rotary, mode):
    """The tangent of a rotated dual tensor is the rotated tangent, of either or both."""
    q, k, tq, tk = _rows(), _rows(1, 1), _rows(2, 2), _rows(1, 3)
    with forward_ad.dual_level(), mode():
        for dq, dk in ((1, 1), (1, 0), (0, 1)):
            x = forward_ad.make_dual(q, tq) if dq else q
            y = forward_ad.make_dual(k, tk) if dk else k
            for out, base, t, dual in zip(rotary(POS, x, y), (q, k), (tq, tk), (dq, dk)):
                p, d = forward_ad.unpack_dual(out)
                _near(p, _turned(base))
                if dual:
                    _near(d, _turned(t))
                else:
                    assert d is None or not d.any()
        p, d = forward_ad.unpack_dual(rotary(POS, forward_ad.make_dual(k, tk)))
        _near(p, _turned(k)), _near(d, _turned(tk))
        assert forward_ad.unpack_dual(rotary(POS, q)).tangent is None
        with pytest.raises(ValueError, match="inplace"):
            rotary(POS, forward_ad.make_dual(q, tq), inplace=True)
        with pytest.raises(ValueError, match="inplace"):
            rotary(POS, q, forward_ad.make_dual(k, tk), inplace=True)


def test_forward_over_backward(rotary):
    """The tangent of a gradient: of the dual gradient of the outputs."""
    q = _rows().requires_grad_()
    g, tg = _rows(2, 4), _rows(2, 5)
    with forward_ad.dual_level():
        (dq,) = torch.autograd.grad(rotary(POS, q), (q,), forward_ad.make_dual(g, tg))
        p, d = forward_ad.unpack_dual(dq)
        _near(p.detach(), _turned(g, True))
        _near(d, _turned(tg, True))


def test_backward_over_forward(rotary):
    """The gradient of a tangent."""
    q, tq, g = _rows(), _rows(2, 2).requires_grad_(), _rows(2, 3)
    with forward_ad.dual_level():
        d = forward_ad.unpack_dual(rotary(POS, forward_ad.make_dual(q, tq))).tangent
        _near(d.detach(), _turned(tq.detach()))
        (dt,) = torch.autograd.grad(d, (tq,), g)
    _near(dt, _turned(g, True))


def test_gradients_as_before(rotary):
    """Backward of both, of one, of a second order; outputs of inputs that need none need none."""
    q, k = _rows().requires_grad_(), _rows(1, 1).requires_grad_()
    gq, gk = _rows(2, 2).requires_grad_(), _rows(1, 3)
    dq, dk = torch.autograd.grad(rotary(POS, q, k), (q, k), (gq, gk), create_graph=True)
    _near(dq.detach(), _turned(gq.detach(), True)), _near(dk, _turned(gk, True))
    h = _rows(2, 6)
    (dg,) = torch.autograd.grad(dq, (gq,), h)
    _near(dg, _turned(h))
    yq, yk = rotary(POS, q.detach(), k)
    assert not yq.requires_grad and yk.requires_grad
    (dk,) = torch.autograd.grad(yk, (k,), gk)
    _near(dk, _turned(gk, True))


def test_function_transforms_are_refused(rotary):
    q = _rows()
    for call in (lambda: torch.func.jvp(lambda x: rotary(POS, x), (q,), (q,)),
                 lambda: torch.func.grad(lambda x: rotary(POS, x).sum())(q),
                 lambda: torch.func.vmap(lambda x: rotary(POS, x))(q[None])):
        with pytest.raises(RuntimeError):
            call()


def _traces():
    from torch.fx.experimental.proxy_tensor import make_fx
    return [lambda f, *a: make_fx(f)(*a), lambda f, *a: make_fx(f, tracing_mode="fake")(*a),
            lambda f, *a: torch.jit.trace(f, a, check_trace=False),
            lambda f, *a: torch.export.export(_Module(f), a, strict=False)]


class _Module(torch.nn.Module):
    def __init__(self, f):
        super().__init__()
        self.f = f

    def forward(self, *a):
        return self.f(*a)


@pytest.mark.parametrize("trace", range(4))
def test_traced_calls_are_refused(rotary, cache, trace):
    """A traced program would hold the output's allocation alone."""
    trace = _traces()[trace]
    table, lengths = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q, k = _rows(4), _rows()
    for f in (lambda q, k: rotary(POS, q, k)[0] + 1,
              lambda q, k: rotary(POS, q.clone(), inplace=True) + 1,
              lambda q, k: cache.attend(q, table, lengths) + 1,
              lambda q, k: cache.step(q, k, k, table, lengths) + 1,
              lambda q, k: (cache.append(k, k, table, lengths), q + 1)[1]):
        with pytest.raises(RuntimeError, match="cannot be traced|data pointer"):
            trace(f, q, k)
    assert rotary._handle.calls == 0


def test_compiled_calls_run(rotary):
    """torch.compile leaves the call between its graphs."""
    q = _rows()
    f = torch.compile(lambda q: rotary(POS, q * 2) + 1, backend="eager")
    _near(f(q) - 1, _turned(q * 2))
    _near(f(q + 1) - 1, _turned((q + 1) * 2))


def test_other_modes_run(rotary):
    """A dispatch mode that records nothing is no trace."""
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):
        _near(rotary(POS, _rows()), _turned(_rows()))


def test_queries_that_overlap_get_an_output_of_rows(cache):
    """Windows over one row of values: like them, an output would hold its rows' values apart."""
    table, lengths = torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    q = torch.arange(64.0).as_strided((4, 2, 8), (1, 8, 1))
    assert torch.empty_like(q).stride(2) != 1
    seen = []
    cache._handle.attend = lambda *a: seen.append(a)
    out = cache.attend(q, table, lengths)
    assert out.shape == q.shape and out.is_contiguous()
    assert seen[0][3:7] == (8 * 4, 1 * 4, 8 * 4, 16 * 4)  # bytes between heads and sequences
