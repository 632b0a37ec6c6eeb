"""Pages of 4-bit values (PagedCache4, adaptq_paged4_*): codes against the rule in 64 bits, value
by value, and attention over the values as they are held against the formula."""
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
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache4
    from adaptq_amd.rotary import Rotary
    globals().update(PagedCache4=PagedCache4, Rotary=Rotary)


def held(x):
    """Rows as 4 bits hold them, in 64 bits."""
    y = x.detach().cpu().double().reshape(-1, 32)
    top = y.abs().amax(1, keepdim=True)
    finite = torch.isfinite(top)
    power = torch.full_like(top, 2.0 ** -125)
    for e in range(-125, 126):  # the smallest that is enough, at most 2^125
        power = torch.where((top > 6 * 2.0 ** (e - 1)) & (e > -125), 2.0 ** e, power)
    a = (y / power).abs()
    best, best_off = torch.zeros_like(a), a.clone()
    for i, point in enumerate(GRID):
        off = (a - point).abs()
        nearer = (off < best_off) | ((off == best_off) & (i % 2 == 0))
        best, best_off = torch.where(nearer, point, best), torch.where(nearer, off, best_off)
    z = torch.where(finite, torch.copysign(best, y) * power, float("nan"))
    return z.reshape(x.shape)


class Case:
    """Sequences whose rows are appended as they come (the keys already turned)."""

    def __init__(self, lengths, heads, group, dim, ps, dtype, *, rot=0, seed=0, extra=1, rows=True):
        self.p = p = S.Pool(lengths, heads, dim, ps, dtype, seed=seed, rows=False, extra=extra)
        k, v = (torch.randint(0, 256, (p.pages, heads, ps, 17 * dim // 32), dtype=torch.uint8,
                              generator=p.g).cuda() for _ in range(2))  # anything
        self.plain = PagedCache4(k, v, dtype=dtype)
        self.cache = PagedCache4(k, v, dtype=dtype, rotary=Rotary(rot)) if rot else self.plain
        self.rot, self.zero = rot, torch.zeros_like(p.lengths)
        self.q = p.normal(len(lengths), heads * group, dim).cuda()
        if rows:
            self.k_in, self.v_in = (p.normal(sum(lengths), heads, dim) for _ in range(2))
            self.offsets = S.spans(lengths)
            self.plain.append(self.k_in.cuda(), self.v_in.cuda(), p.table, self.zero, self.offsets)
            at = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
            k, v = held(self.k_in), held(self.v_in)
            self.k, self.v = ([x[a:b] for a, b in zip(at, at[1:])] for x in (k, v))

    def want(self, *, scale=None, window=None, softcap=None, slopes=None, prefix=None, first=None,
             extra=0):
        p = self.p
        outs, tols = [], []
        for i in range(len(p.held)):
            n = self.k[i].shape[0]
            q, err = self.q[i:i + 1].cpu().double(), None
            if self.rot and n:
                q, err = R.rotate(self.q[i:i + 1].float(), torch.tensor([n - 1]), self.rot)
            at = torch.tensor([n - 1])
            seen = S.sees(n, at, torch.zeros(1) if first is None else first[i:i + 1],
                          torch.zeros(1) if prefix is None else prefix[i:i + 1], window)
            # (products of three bf16 numbers, whatever the queries' type: fp32's tolerance, then
            # the rounding to the type)
            o, t, _, _ = S.attend(q, self.k[i].transpose(0, 1), self.v[i].transpose(0, 1), seen, at,
                                  1 / math.sqrt(p.dim) if scale is None else scale, torch.float32,
                                  softcap=softcap, slopes=slopes, q_err=err)
            outs.append(o)
            tols.append(t + R.u(p.dtype) * o.abs() + R._tiny(p.dtype))
        return torch.cat(outs), torch.cat(tols)

    def check(self, **kw):
        gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        got = self.cache.attend(self.q, self.p.table, self.p.lengths, **gpu)
        R.check(got, *self.want(**kw))
        return got


# ---------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("heads,ps", [(1, 16), (3, 48)])
def test_append_and_read(dtype, dim, heads, ps):
    lengths = [0, 1, 3, 4, 5, 16, 17, 33, 100]
    c = Case(lengths, heads, 1, dim, ps, dtype, seed=dim)
    k, v = c.plain.read(sum(lengths), c.p.table, c.zero, c.offsets)
    assert k.dtype == torch.float32
    assert torch.equal(k.cpu().double(), held(c.k_in)) and torch.equal(v.cpu().double(), held(c.v_in))
    # behind what is there: one token a sequence
    a, b = c.p.normal(9, heads, dim), c.p.normal(9, heads, dim)
    c.plain.append(a.cuda(), b.cuda(), c.p.table, c.p.lengths)
    k2, v2 = c.plain.read(9, c.p.table, c.p.lengths)
    assert torch.equal(k2.cpu().double(), held(a)) and torch.equal(v2.cpu().double(), held(b))
    again = c.plain.read(sum(lengths), c.p.table, c.zero, c.offsets)
    assert torch.equal(again[0], k) and torch.equal(again[1], v)  # what was there stays


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_rounding(dtype):
    """Values on the points, between them and beside the middles, at scales over the type's range;
    zeros of both signs; blocks of zeros."""
    info = torch.finfo(dtype)
    points = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0]
    base = torch.tensor(points, dtype=torch.float64)
    near = torch.cat([base, base * (1 + info.eps), base * (1 - info.eps / 2)])
    rows = []
    for e in range(-130, 128, 3):
        x = near * 2.0 ** e
        for top in (6.0, 5.5, 3.1, 3.0, 4.0):
            for part in x.split(15):
                y = torch.zeros(32, dtype=torch.float64)
                part = part.clamp(max=top * 2.0 ** e)
                y[:15], y[15:30], y[30] = part, -part, top * 2.0 ** e
                y[31] = -0.0
                rows.append(y)
    x = torch.stack(rows)
    x = x.clamp(-info.max, info.max).to(dtype)
    x = torch.cat([x, torch.zeros(1, 32, dtype=dtype), torch.full((1, 32), info.max, dtype=dtype),
                   torch.full((1, 32), info.smallest_normal, dtype=dtype)])
    n = x.shape[0]
    x = x.view(n, 1, 32)
    c = Case([n], 1, 1, 32, 64, dtype, rows=False)
    off = S.spans([n])
    c.plain.append(x.cuda(), x.flip(0).cuda(), c.p.table, c.zero, off)
    k, v = c.plain.read(n, c.p.table, c.zero, off)
    assert torch.equal(k.cpu().double(), held(x))
    assert torch.equal(v.cpu().double(), held(x.flip(0)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(dtype):
    """A block with one reads as NaN, its neighbours as ever."""
    x = torch.randn(3, 2, 96, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0, 1, 40], x[1, 0, 0], x[2, 1, 95] = float("inf"), float("nan"), -float("inf")
    c = Case([3], 2, 1, 96, 16, dtype, rows=False)
    off = S.spans([3])
    c.plain.append(x.cuda(), x.cuda(), c.p.table, c.zero, off)
    want = held(x)
    assert torch.isnan(want).sum() == 96
    for y in c.plain.read(3, c.p.table, c.zero, off):
        assert torch.equal(torch.isnan(y).cpu(), torch.isnan(want))
        assert torch.equal(y.cpu().double().nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot,interleaved,dim", [(64, False, 64), (64, True, 128), (20, False, 96),
                                                 (6, True, 32), (256, False, 256), (128, False, 128)])
def test_rotated_keys(dtype, rot, interleaved, dim):
    """As the same rows turned by Rotary and appended without."""
    lengths = [3, 50, 0, 77]
    rotary = Rotary(rot, interleaved=interleaved)
    a, b = Case(lengths, 2, 1, dim, 16, dtype, rows=False), Case(lengths, 2, 1, dim, 16, dtype, rows=False)
    k, v = a.p.normal(130, 2, dim).cuda(), a.p.normal(130, 2, dim).cuda()
    off = S.spans(lengths)
    start = torch.tensor([0, 5, 0, 1000], dtype=torch.int32).cuda() * 0
    PagedCache4(a.plain.k_pages, a.plain.v_pages, dtype=dtype, rotary=rotary).append(
        k, v, a.p.table, start, off)
    at = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).cuda()
    b.plain.append(rotary(at, k), v, b.p.table, start, off)
    for x, y in zip(a.plain.read(130, a.p.table, start, off), b.plain.read(130, b.p.table, start, off)):
        assert torch.equal(x, y)


def test_places_that_are_not_there():
    """Tokens outside the offsets, positions without a page, negative lengths: left out; read as
    zeros; nothing else changes."""
    c = Case([40, 40, 40], 2, 1, 64, 16, torch.bfloat16)
    before = [x.clone() for x in (c.plain.k_pages, c.plain.v_pages)]
    table = c.p.table.clone()
    table[0, 2], table[1, :] = -1, 2 ** 31 - 1
    lengths = torch.tensor([32, 0, -5], dtype=torch.int32).cuda()
    k = c.p.normal(30, 2, 64).cuda()
    off = torch.tensor([4, 12, 20, 25], dtype=torch.int32).cuda()
    c.plain.append(k, k, table, lengths, off)
    assert all(torch.equal(a, b) for a, b in zip(before, (c.plain.k_pages, c.plain.v_pages)))
    for x in c.plain.read(30, table, lengths, off):
        assert (x == 0).all()
    for off in ([0, 2 ** 31 - 1, -4, 7], [-9, -9, 5, 2 ** 31 - 1], [30, 20, 10, 0]):
        c.plain.append(k, k, torch.full_like(table, -1), lengths, torch.tensor(off, dtype=torch.int32).cuda())
    assert all(torch.equal(a, b) for a, b in zip(before, (c.plain.k_pages, c.plain.v_pages)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows(dtype):
    """Rows off 16 bytes, parts of one projection."""
    x = torch.randn(70, 9, 67, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    c = Case([70], 2, 1, 64, 16, dtype, rows=False)
    off = S.spans([70])
    for pad in (0, 1, 3):
        k, v = x[:, 2:4, pad:pad + 64], x[:, 5:7, pad:pad + 64]
        c.plain.append(k, v, c.p.table, c.zero, off)
        a, b = c.plain.read(70, c.p.table, c.zero, off)
        assert torch.equal(a.cpu().double(), held(k)) and torch.equal(b.cpu().double(), held(v))


def test_many_tokens():
    """Blocks of many tokens, more than one round of a block's threads."""
    for heads, dim, n in ((8, 128, 5000), (1, 32, 9000), (14, 256, 2500)):
        c = Case([n, 7], heads, 1, dim, 64, torch.bfloat16, seed=n)
        k, v = c.plain.read(n + 7, c.p.table, c.zero, c.offsets)
        assert torch.equal(k.cpu().double(), held(c.k_in))
        assert torch.equal(v.cpu().double(), held(c.v_in))


# ---------------------------------------------------------------- attention

EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 700, 0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("heads,group,ps", [(2, 1, 16), (1, 4, 48), (1, 5, 16)])
def test_lengths(dtype, dim, heads, group, ps):
    Case(EDGES, heads, group, dim, ps, dtype, seed=dim).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 3), (2, 4), (2, 7), (1, 16), (2, 17),
                                         (1, 40), (14, 3)])
def test_groups(dtype, dim, heads, group):
    Case([5, 100, 0, 333], heads, group, dim, 32, dtype, seed=group).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 4, 8])
@pytest.mark.parametrize("lengths,ps", [([20000], 64), ([9000, 1, 700], 16), ([5000, 4097], 256)])
def test_long(dtype, group, lengths, ps):
    c = Case(lengths, 2, group, 128, ps, dtype)
    got = c.check()
    assert torch.equal(c.check(), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [3, 6])
@pytest.mark.parametrize("window", [None, 1, 31, 100, 500])
def test_masks_caps_and_biases(dtype, group, window):
    lengths = [0, 1, 33, 100, 640, 2000]
    c = Case(lengths, 2, group, 64, 16, dtype)
    n = len(lengths)
    g = torch.Generator().manual_seed(4)
    first = torch.randint(-3, 60, (n,), generator=g).int()
    prefix = torch.randint(-3, 90, (n,), generator=g).int()
    c.check(window=window, first=first)
    c.check(window=window, prefix=prefix, softcap=20.0)
    c.check(window=window, first=first, prefix=prefix, slopes=torch.rand(2 * group))
    c.check(window=window, scale=-0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [3, 6])
@pytest.mark.parametrize("slope", [0.03, 0.045, 0.052])
def test_weights_at_the_end_of_fp32(dtype, group, slope):
    """A token of its own, whose values are 0 in some channels, and a prefix 1,900 tokens away: e^-57
    to e^-104 of the weight."""
    lengths = [2000, 1950]
    c = Case(lengths, 2, group, 64, 16, dtype)
    c.check(window=1, prefix=torch.full((2,), 70, dtype=torch.int32),
            slopes=slope * torch.linspace(1, 1.05, 2 * group))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotated_queries(dtype):
    Case([1, 50, 700, 0], 2, 4, 128, 16, dtype, rot=128).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [2, 5])
def test_nan_that_is_not_seen(dtype, group):
    """Stale bytes behind the tokens (the pools begin with any), and NaN that a mask hides."""
    c = Case([100, 45], 2, group, 64, 16, dtype)
    kw = dict(window=20, prefix=torch.full((2,), 5, dtype=torch.int32).cuda())
    clean = c.cache.attend(c.q, c.p.table, c.p.lengths, **kw)
    for x in (c.k_in, c.v_in):
        x[6:80] = float("nan")
        x[106:124] = float("inf")
    c.plain.append(c.k_in.cuda(), c.v_in.cuda(), c.p.table, c.zero, c.offsets)
    assert torch.equal(c.cache.attend(c.q, c.p.table, c.p.lengths, **kw), clean)
    assert torch.isnan(c.cache.attend(c.q, c.p.table, c.p.lengths)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot", [0, 64])
@pytest.mark.parametrize("group,dim", [(3, 64), (4, 128), (7, 96)])
def test_step(dtype, rot, group, dim):
    """Append and attention in one: the bytes and outputs of the two calls."""
    lengths = [0, 1, 31, 64, 100, 700]
    c = Case(lengths, 2, group, dim, 16, dtype, rot=rot)
    n = len(lengths)
    k, v = c.p.normal(n, 2, dim).cuda(), c.p.normal(n, 2, dim).cuda()
    other = PagedCache4(c.plain.k_pages.clone(), c.plain.v_pages.clone(), dtype=dtype,
                        rotary=Rotary(rot) if rot else None)
    got = c.cache.step(c.q, k, v, c.p.table, c.p.lengths)
    other.append(k, v, c.p.table, c.p.lengths)
    assert torch.equal(other.k_pages, c.cache.k_pages)
    assert torch.equal(other.v_pages, c.cache.v_pages)
    assert torch.equal(got, other.attend(c.q, c.p.table, c.p.lengths + 1))
    first = torch.full((n,), 10 ** 6, dtype=torch.int32).cuda()  # nothing is seen: still appended
    got = c.cache.step(c.q, v, k, c.p.table, c.p.lengths, first=first)
    other.append(v, k, c.p.table, c.p.lengths)
    assert (got == 0).all() and torch.equal(other.k_pages, c.cache.k_pages)
    assert torch.equal(other.v_pages, c.cache.v_pages)


def test_offsets_beyond_32_bits():
    """Pools of more than 2^31 bytes, their last pages used."""
    pages, heads, ps, dim = 70000, 8, 64, 128
    cache = PagedCache4.allocate(pages, heads, ps, dim)
    assert cache.k_pages.numel() > 2 ** 31
    c = Case([300], heads, 4, dim, ps, torch.bfloat16)
    c.p.table_host[0, :5] = torch.tensor([69999, 3, 65536, 69998, 40000], dtype=torch.int32)
    c.p.table.copy_(c.p.table_host[:, :c.p.table.shape[1]])
    cache.append(c.k_in.cuda(), c.v_in.cuda(), c.p.table, c.zero, c.offsets)
    k, v = cache.read(300, c.p.table, c.zero, c.offsets)
    assert torch.equal(k.cpu().double(), held(c.k_in)) and torch.equal(v.cpu().double(), held(c.v_in))
    c.cache = cache
    c.check()


def test_captured_and_replayed():
    c = Case([100, 333], 2, 4, 128, 64, torch.bfloat16, extra=20)
    k, v = c.p.normal(2, 2, 128).cuda(), c.p.normal(2, 2, 128).cuda()
    lengths, out = c.p.lengths.clone(), torch.empty_like(c.q)

    def step():
        c.cache.step(c.q, k, v, c.p.table, lengths, out=out)
        lengths.add_(1)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lengths.copy_(c.p.lengths)
    got = []
    for _ in range(5):
        graph.replay()
        got.append(out.clone())
        (torch.randn(1000, device="cuda") @ torch.randn(1000, device="cuda")).item()
    lengths.copy_(c.p.lengths)
    for x in got:
        step()
        assert torch.equal(out, x)


def test_streams():
    """Rows appended on one stream, read on another: the cache orders them."""
    c = Case([3000, 2000], 4, 4, 128, 64, torch.bfloat16)
    want = c.cache.attend(c.q, c.p.table, c.p.lengths)
    k, v = c.k_in.cuda(), c.v_in.cuda()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        c.plain.k_pages.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            c.cache.append(k, v, c.p.table, c.zero, c.offsets)
        with torch.cuda.stream(b):
            got = c.cache.attend(c.q, c.p.table, c.p.lengths)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals():
    c = Case([10, 20], 2, 2, 64, 16, torch.float16)
    q, t, n = c.q, c.p.table, c.p.lengths
    k = q[:, :2]
    with pytest.raises(ValueError):
        PagedCache4.allocate(4, 2, 16, 40)
    with pytest.raises(RuntimeError):
        PagedCache4.allocate(4, 2, 16, 288)
    with pytest.raises(RuntimeError):
        PagedCache4.allocate(4, 2, 24, 64)
    u8 = torch.zeros(4, 2, 16, 34, dtype=torch.uint8, device="cuda")
    for a, b, kw in ((u8.int(), u8.int(), {}), (u8, u8[:2], {}), (u8[..., :33], u8[..., :33], {}),
                     (u8.cpu(), u8.cpu(), {}), (u8, u8.clone(), dict(dtype=torch.float64))):
        with pytest.raises((ValueError, TypeError)):
            PagedCache4(a, b, **kw)
    with pytest.raises(RuntimeError):
        PagedCache4(u8, u8)  # one pool twice
    for call in (lambda: c.cache.attend(q.float(), t, n), lambda: c.cache.attend(q, t, n, softcap=-1.0),
                 lambda: c.cache.attend(q, t, n, window=0), lambda: c.cache.append(k, k, t, n[:1]),
                 lambda: c.cache.append(k[:1], k, t, n), lambda: c.cache.read(3, t, n),
                 lambda: c.cache.step(q, k[:1], k[:1], t, n),
                 lambda: c.cache.attend(q, t, n, first=torch.zeros(3, dtype=torch.int32).cuda())):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(RuntimeError):
        c.cache.attend(q[:, :3], t, n)
    with pytest.raises(RuntimeError):
        c.cache.attend(q, t, n, out=q)


def test_handles_of_the_other_kind():
    """An exact cache's handle is refused by the 4-bit calls, and the other way about."""
    from adaptq_amd.paged import PagedCache  # noqa: F401
    x = torch.zeros(2, 1, 16, 64, device="cuda")
    y = torch.zeros(2, 1, 16, 64, device="cuda")
    u = [torch.zeros(2, 1, 16, 34, dtype=torch.uint8, device="cuda") for _ in range(2)]
    a = L.adaptq_paged_create(x.data_ptr(), y.data_ptr(), 2, 16, 1, 64, 0, None)
    b = L.adaptq_paged4_create(u[0].data_ptr(), u[1].data_ptr(), 2, 16, 1, 64, 0, None)
    assert a and b
    seqs = (None, 0, 0, None, 0)
    assert L.adaptq_paged4_append_device(a, None, None, 0, 0, 0, 0, 0, *seqs, None, None) == -1
    assert b"exact" in L.adaptq_last_error()
    assert L.adaptq_paged4_read_device(a, None, None, 0, *seqs, None, None) == -1
    assert L.adaptq_paged_append_device(b, None, None, 0, 0, 0, 0, 0, *seqs, None, None) == -1
    assert b"4-bit" in L.adaptq_last_error()
    assert L.adaptq_paged_prompt_device(b, None, None, 1, 0, 0, 0, 0, 0, *seqs, None, 0.0, None, None,
                                        0, None) == -1
    assert L.adaptq_paged_evict_device(b, None, 0, 0, *seqs, 1, 0, None, 0, 0, None, None) == -1
    assert L.adaptq_paged4_attend_device(b, None, None, 1, 0, 0, 0, 0, *seqs, 0.0, None, None) == 0
    sc = _lib.Scores(-2.0, 0, None, None, None)
    assert L.adaptq_paged4_attend_device(b, None, None, 1, 0, 0, 0, 0, *seqs, 0.0, C.byref(sc), None) == -1
    L.adaptq_paged_destroy(a)
    L.adaptq_paged4_destroy(b)
    L.adaptq_paged4_destroy(None)
