"""The paged cache (adaptq_paged_*, adaptq_amd.paged) against the formulas in 64 bits:
appends bit for bit where nothing is rounded, attention over every type, head layout and
length at which it can go wrong, pages that hold anything behind the tokens, tables that
name no page, strides, windows, streams, graphs, pools beyond 32-bit offsets, refusals."""
import ctypes as C
import math
import random

import pytest
import torch

import paged_ref as R
from adaptq_amd import _lib

pytestmark = pytest.mark.gpu
L = _lib.lib
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    globals().update(PagedCache=PagedCache, Rotary=Rotary)


class Server:
    """Sequences over a pool: their tables, lengths and rows as the 64-bit side sees them."""

    def __init__(self, lengths, heads, dim, page_size, dtype, rot=0, seed=0, spare=3, room=1,
                 fill=float("nan"), pools=None, **kw):
        self.g = torch.Generator().manual_seed(seed)
        self.heads, self.dim, self.ps, self.dtype = heads, dim, page_size, dtype
        self.rot, self.kw = rot, kw
        need = [-(-(n + room) // page_size) for n in lengths]
        pages = sum(need) + spare
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        width = max(need) + 1
        # entries behind a sequence's pages hold anything
        table = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(lengths), width + 2), generator=self.g,
                              dtype=torch.int64).int()
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = torch.tensor(order[at:at + n])
            at += n
        self.free = order[at:]
        self.table_host, self.held = table, list(lengths)
        self.table = table.cuda()[:, :width]  # rows further apart than they are wide
        self.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
        shape = (pages, heads, page_size, dim)
        kp, vp = pools or (torch.full(shape, fill, dtype=dtype, device="cuda") for _ in range(2))
        rotary = Rotary(rot, **kw) if rot else None
        self.cache = PagedCache(kp, vp, rotary=rotary)
        self.k, self.v = [], []
        for i, n in enumerate(lengths):  # rows as the pages hold them (keys already rotated)
            k, v = self.normal(n, heads, dim), self.normal(n, heads, dim)
            self.k.append(k)
            self.v.append(v)
            self.put(i, 0, k, v)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dtype)

    def place(self, i, first, n):
        p = torch.arange(first, first + n)
        return self.table_host[i, p // self.ps].long().cuda(), (p % self.ps).cuda()

    def put(self, i, first, k, v):
        page, slot = self.place(i, first, k.shape[0])
        self.cache.k_pages[page, :, slot] = k.cuda()
        self.cache.v_pages[page, :, slot] = v.cuda()

    def want(self, q, n_tokens=None, scale=None, window=None, extra=0):
        """(out, tolerance) [sequences, q_heads, dim] in 64 bits; q as given to attend."""
        outs, tols = [], []
        for i, (k, v) in enumerate(zip(self.k, self.v)):
            n = k.shape[0]
            lo = max(0, n - window) if window else 0
            x, err = q[i:i + 1].cpu().double(), 0.0
            if self.rot and n:
                x, err = R.rotate(q[i:i + 1].float(), torch.tensor([n - 1]), self.rot, **self.kw)
                err = err[0].view(self.heads, -1, self.dim)
            o, t = R.attend(x[0].view(self.heads, -1, self.dim), k[lo:].transpose(0, 1),
                            v[lo:].transpose(0, 1),
                            scale if scale is not None else 1 / math.sqrt(self.dim), self.dtype,
                            err)
            outs.append(o.reshape(-1, self.dim))
            tols.append(t.reshape(-1, self.dim))
        return torch.stack(outs), torch.stack(tols)

    def queries(self, q_heads):
        return self.normal(len(self.held), q_heads, self.dim).cuda()

    def attend(self, q, **kw):
        return self.cache.attend(q, self.table, self.lengths, **kw)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 0]


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("heads,group,ps", [(2, 1, 16), (1, 4, 48)])
def test_lengths(dtype, dim, heads, group, ps):
    s = Server(EDGES, heads, dim, ps, dtype, seed=dim)
    q = s.queries(heads * group)
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 7), (1, 16), (2, 17), (1, 71), (14, 3)])
def test_groups(dtype, dim, heads, group):
    s = Server([5, 100, 0, 333], heads, dim, 32, dtype, seed=group)
    q = s.queries(heads * group)
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps,lengths", [
    (16, [20000]), (64, [5000, 1, 9000]), (256, [4097] * 3), (4096, [3000, 8191]),
    (176, [7000, 0, 0, 2500]), (65536, [70000]),
])
def test_long(dtype, ps, lengths):
    """Few sequences: split over their length and joined."""
    s = Server(lengths, 2, 64, ps, dtype, seed=len(lengths))
    q = s.queries(8)
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group,lengths", [
    (128, 1, [40000]), (128, 16, [2176]), (128, 16, [2177]), (128, 17, [9000]), (128, 3, [33000]),
    (64, 16, [3000, 20000]), (256, 8, [5000]), (256, 16, [30000]), (80, 5, [8000, 1, 8000]),
])
def test_one_key_head(dtype, dim, group, lengths):
    """Hundreds of pieces of one segment, joined by groups first."""
    s = Server(lengths, 1, dim, 64, dtype, seed=group)
    q = s.queries(group)
    first = s.attend(q)
    R.check(first, *s.want(q))
    assert torch.equal(s.attend(q), first)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 63, 64, 65, 300, 1000])
def test_many_sequences(dtype, n):
    rng = random.Random(n)
    s = Server([rng.choice((0, 1, 17, rng.randint(0, 150))) for _ in range(n)], 2, 32, 16, dtype,
               seed=n)
    q = s.queries(4)
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000, 2 ** 31 - 1])
def test_window(dtype, window):
    s = Server([0, 1, 33, 100, 101, 640, 2000], 2, 64, 16, dtype, seed=window % 97)
    q = s.queries(6)
    R.check(s.attend(q, window=window), *s.want(q, window=window))


@pytest.mark.parametrize("scale", [1.0, 0.01, -0.5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scale(dtype, scale):
    s = Server([40, 200], 2, 64, 16, dtype)
    q = s.queries(4)
    R.check(s.attend(q, scale=scale), *s.want(q, scale=scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot,interleaved,dim", [(64, False, 64), (64, True, 128), (20, False, 80),
                                                 (6, True, 8), (256, False, 256)])
def test_rotated_queries(dtype, rot, interleaved, dim):
    s = Server([0, 1, 50, 700], 2, dim, 16, dtype, rot=rot, interleaved=interleaved,
               scaling="yarn", factor=4.0, context=512)
    q = s.queries(6)
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_and_values(dtype):
    """Scores in the hundreds (weights that all but vanish), a rotated fp16 query at the top of
    its range, and values near the type's largest."""
    s = Server([300], 1, 64, 16, dtype, rot=64)
    big = 30000.0 if dtype == torch.float16 else 1e30
    s.k[0][:, :, 5] *= 40
    s.v[0][:, 0, 7] = big
    s.put(0, 0, s.k[0], s.v[0])
    q = s.queries(4)
    q[0, 1] *= 20
    q[0, 2, :] = 65000.0 if dtype == torch.float16 else 1e4
    R.check(s.attend(q, scale=0.125), *s.want(q, scale=0.125))
    q = s.queries(4) * 1e-3
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(dtype):
    """In a token of one head they reach that head's queries as the formula says, and no other."""
    s = Server([100, 100, 100], 2, 64, 16, dtype)
    q = s.queries(4)
    clean = s.attend(q)
    k, v = s.k, s.v
    v[0][40, 0, 3] = float("nan")
    v[1][99, 1, 9] = float("inf")
    k[2][7, 0, 0] = float("nan")
    for i in range(3):
        s.put(i, 0, k[i], v[i])
    got = s.attend(q)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :2, 3] = bad[2, :2] = True
    assert torch.isnan(got[bad]).all()
    bad[1, 2:, 9] = True
    assert torch.isinf(got[1, 2:, 9]).all()
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity(dtype):
    """A key that scores minus infinity has no weight; only such keys: a softmax of nothing but
    zeros, NaN as the formula has it."""
    s = Server([100, 40], 1, 64, 16, dtype)
    q = s.queries(2).abs() + 0.01
    s.k[0][10:60, :, 0] = -float("inf")
    s.k[1][:, :, 0] = -float("inf")
    for i in range(2):
        s.put(i, 0, s.k[i], s.v[i])
    got = s.attend(q)
    keep = torch.cat((torch.arange(10), torch.arange(60, 100)))
    s.k[0], s.v[0] = s.k[0][keep], s.v[0][keep]
    s.k[1], s.v[1] = s.k[1][:0], s.v[1][:0]
    want, tol = s.want(q)
    R.check(got[:1], want[:1], tol[:1])
    assert torch.isnan(got[1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_a_page_are_left_out(dtype):
    s = Server([200, 70, 33, 20], 2, 64, 16, dtype)
    q = s.queries(4)
    t = s.table_host
    t[0, 3], t[0, 12] = -1, 10 ** 9       # tokens 48-63 and 192-199
    t[1, :] = 2 ** 31 - 1                 # none at all
    s.table.copy_(t[:, :s.table.shape[1]])
    s.lengths[2] = 10 ** 6                # more than the table is wide
    s.lengths[3] = -5
    width = s.table.shape[1] * 16
    keep = [i for i in range(200) if i // 16 not in (3, 12)]
    s.k[0], s.v[0] = s.k[0][keep], s.v[0][keep]
    s.k[1], s.v[1] = s.k[1][:0], s.v[1][:0]
    s.k[3], s.v[3] = s.k[3][:0], s.v[3][:0]
    t[2, 3:] = -7                         # sequence 2: 33 tokens in 3 pages, then nothing
    s.table.copy_(t[:, :s.table.shape[1]])
    page, slot = s.place(2, 33, 15)
    more = s.normal(15, 2, 64), s.normal(15, 2, 64)
    s.put(2, 33, *more)
    s.k[2], s.v[2] = torch.cat((s.k[2], more[0])), torch.cat((s.v[2], more[1]))
    assert width > 48
    R.check(s.attend(q), *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_run_without_pages(dtype):
    """Whole pieces of a cut sequence have no page: 4,000 tokens in the middle, or all."""
    s = Server([6000, 6000], 1, 64, 16, dtype)
    q = s.queries(4)
    s.table_host[0, 50:300] = -1
    s.table_host[1, :] = 2 ** 31 - 1
    s.table.copy_(s.table_host[:, :s.table.shape[1]])
    keep = [*range(800), *range(4800, 6000)]
    s.k[0], s.v[0] = s.k[0][keep], s.v[0][keep]
    s.k[1], s.v[1] = s.k[1][:0], s.v[1][:0]
    R.check(s.attend(q), *s.want(q))


def test_table_of_no_width():
    s = Server([0, 0], 1, 64, 16, torch.float32)
    q = s.queries(2)
    s.lengths[:] = 100
    out = s.cache.attend(q, s.table[:, :0], s.lengths)
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_queries_and_outputs(dtype):
    """Queries that are part of a projection, rows off 16 bytes, an output with room around it."""
    s = Server([30, 0, 170], 2, 64, 16, dtype)
    q = s.queries(4)
    want = s.want(q)
    for pad in (0, 1, 8):
        wide = torch.full((3, 9, 64 + pad), 7.0, dtype=dtype, device="cuda")
        wide[:, 2:6, pad:] = q
        room = torch.full((4, 6, 64 + pad), 5.0, dtype=dtype, device="cuda")
        out = room[:3, 1:5, pad:]
        got = s.attend(wide[:, 2:6, pad:], out=out)
        assert got is out
        R.check(out, *want)
        out.fill_(5.0)
        assert (room == 5.0).all()  # nothing around the rows was written
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    R.check(s.attend(q2), *want)


def test_equal_calls_give_equal_bits():
    s = Server([5000, 77, 0, 1234, 4096], 4, 128, 64, torch.bfloat16)
    q = s.queries(16)
    first = s.attend(q)
    for _ in range(5):
        s.attend(s.queries(16))
        assert torch.equal(s.attend(q), first)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^31 values a side, its last pages used."""
    pages, heads, ps, dim = 70000, 4, 64, 128
    pools = [torch.empty(pages, heads, ps, dim, dtype=torch.bfloat16, device="cuda")
             for _ in range(2)]
    assert pools[0].numel() > 2 ** 31
    s = Server([300, 100], heads, dim, ps, torch.bfloat16, pools=pools, rot=64)
    rows = [s.k[0], s.v[0]]
    s.table_host[0, :5] = torch.tensor([69999, 3, 65536, 69998, 40000], dtype=torch.int32)
    s.table.copy_(s.table_host[:, :s.table.shape[1]])
    s.put(0, 0, *rows)
    q = s.queries(8)
    R.check(s.attend(q), *s.want(q))
    k, v = s.normal(2, heads, dim), s.normal(2, heads, dim)
    s.cache.append(k.cuda(), v.cuda(), s.table, s.lengths)
    page, slot = s.place(0, 300, 1)
    assert page.item() == 40000
    assert torch.equal(pools[1][page, :, slot][0].cpu(), v[0])


# ---------------------------------------------------------------- append

def _appended(s, i, first, k, v, kp, vp):
    """Expected pools after tokens first, first + 1, ... of sequence i; keys with a tolerance."""
    n = k.shape[0]
    page, slot = s.place(i, first, n)
    vp[page, :, slot] = v.cuda()
    want, tol = k.double(), torch.zeros(k.shape, dtype=torch.float64)
    if s.rot:
        want, tol = R.rotate(k, torch.arange(first, first + n), s.rot, **s.kw)
    R.check(s.cache.k_pages[page, :, slot], want, tol, f"sequence {i}")
    kp[page, :, slot] = s.cache.k_pages[page, :, slot]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 0, False), (64, 64, False), (128, 64, True),
                                                 (80, 40, False), (80, 6, True), (8, 2, False),
                                                 (256, 256, True), (96, 96, False)])
def test_append(dtype, dim, rot, interleaved):
    """Prompts of 0, 1, 40 and 17 tokens, then one token a sequence; the rest of the pools as
    it was."""
    kw = dict(interleaved=interleaved, scaling="bands", factor=4.0, context=64) if rot else {}
    s = Server([0, 31, 5, 100], 3, dim, 16, dtype, rot=rot, room=60, fill=3.0, **kw)
    counts = [0, 1, 40, 17]
    k, v = s.normal(60, 3, dim), s.normal(60, 3, dim)  # two rows more than the offsets name
    off = torch.tensor([0, 0, 1, 41, 58], dtype=torch.int32).cuda()
    kp, vp = s.cache.k_pages.clone(), s.cache.v_pages.clone()
    s.cache.append(k.cuda(), v.cuda(), s.table, s.lengths, off)
    at = 0
    for i, n in enumerate(counts):
        _appended(s, i, s.held[i], k[at:at + n], v[at:at + n], kp, vp)
        at += n
    assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)
    s.lengths += torch.tensor(counts, dtype=torch.int32).cuda()
    s.cache.append(k[:4].cuda(), v[:4].cuda(), s.table, s.lengths)
    for i in range(4):
        _appended(s, i, s.held[i] + counts[i], k[i:i + 1], v[i:i + 1], kp, vp)
    assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)


def test_append_many_tokens():
    """Enough tokens that a block takes several, over many sequences, some of them empty."""
    rng = random.Random(5)
    counts = [rng.choice((0, 0, 1, 3, rng.randint(0, 300))) for _ in range(200)]
    s = Server([rng.randint(0, 40) for _ in counts], 2, 64, 32, torch.float16, rot=64, room=300,
               fill=1.0)
    total = sum(counts)
    assert total > 4096
    k, v = s.normal(total, 2, 64), s.normal(total, 2, 64)
    off = [sum(counts[:i]) for i in range(len(counts) + 1)]
    kp, vp = s.cache.k_pages.clone(), s.cache.v_pages.clone()
    s.cache.append(k.cuda(), v.cuda(), s.table, s.lengths, torch.tensor(off).int().cuda())
    for i, n in enumerate(counts):
        if n:
            _appended(s, i, s.held[i], k[off[i]:off[i + 1]], v[off[i]:off[i + 1]], kp, vp)
    assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_strided(dtype):
    for pad in (0, 1, 8):
        s = Server([3, 18], 2, 64, 16, dtype, rot=64, fill=0.0)
        fused = s.normal(2, 9, 64 + pad).cuda()
        k, v = fused[:, 4:6, pad:], fused[:, 6:8, pad:]
        kp, vp = s.cache.k_pages.clone(), s.cache.v_pages.clone()
        s.cache.append(k, v, s.table, s.lengths)
        for i in range(2):
            _appended(s, i, s.held[i], k[i:i + 1].cpu(), v[i:i + 1].cpu(), kp, vp)
        assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)


def test_append_without_a_page():
    """Tokens past the table, on pages outside the pool or of sequences of negative length are
    left out, and so are tokens outside ragged offsets; nothing else changes."""
    s = Server([14, 30, 7, 50], 2, 64, 16, torch.float32, fill=2.0)
    s.table_host[1, 1] = -1
    s.table_host[3, :] = 10 ** 6
    s.table.copy_(s.table_host[:, :s.table.shape[1]])
    s.lengths[2] = -1
    k, v = s.normal(20, 2, 64), s.normal(20, 2, 64)
    kp, vp = s.cache.k_pages.clone(), s.cache.v_pages.clone()
    off = torch.tensor([2, 6, 10, 12, 16], dtype=torch.int32).cuda()
    s.cache.append(k.cuda(), v.cuda(), s.table[:, :1], s.lengths, off)
    _appended(s, 0, 14, k[2:4], v[2:4], kp, vp)  # tokens 4, 5 lie past a table of one column
    assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)
    off = torch.tensor([0, 0, 2, 2, 2], dtype=torch.int32).cuda()
    s.cache.append(k.cuda(), v.cuda(), s.table, s.lengths, off)  # page -1
    s.lengths[:] = 2 ** 31 - 1
    s.cache.append(k[:4].cuda(), v[:4].cuda(), s.table, s.lengths)
    assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)


def test_shared_pages():
    """Sequences that begin with the same pages (a common prompt) go on in pages of their own."""
    s = Server([32, 40], 2, 64, 16, torch.bfloat16)
    s.table_host[0, :2] = s.table_host[1, :2]
    s.table.copy_(s.table_host[:, :s.table.shape[1]])
    s.k[0], s.v[0] = s.k[1][:32], s.v[1][:32]
    q = s.queries(4)
    R.check(s.attend(q), *s.want(q))
    k, v = s.normal(2, 2, 64), s.normal(2, 2, 64)
    out = s.cache.step(q, k.cuda(), v.cuda(), s.table, s.lengths)
    for i in range(2):
        s.k[i], s.v[i] = torch.cat((s.k[i], k[i:i + 1])), torch.cat((s.v[i], v[i:i + 1]))
    R.check(out, *s.want(q))


# ---------------------------------------------------------------- steps

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,group,dim,rot,ps", [
    (2, 1, 64, 64, 16), (4, 4, 128, 128, 32), (1, 20, 80, 0, 48), (2, 3, 256, 128, 16),
    (3, 2, 40, 8, 16),
])
def test_step_is_append_then_attend(dtype, heads, group, dim, rot, ps):
    lengths = [0, 1, 15, 16, 31, 32, 64, 300, 2000]
    a, b = (Server(lengths, heads, dim, ps, dtype, rot=rot, fill=0.5) for _ in range(2))
    q, (k, v) = a.queries(heads * group), (a.normal(9, heads, dim).cuda() for _ in range(2))
    for window in (None, 20):
        got = a.cache.step(q, k, v, a.table, a.lengths, window=window)
        b.cache.append(k, v, b.table, b.lengths)
        want = b.cache.attend(q, b.table, b.lengths + 1, window=window)
        assert torch.equal(got, want)
        assert torch.equal(a.cache.k_pages, b.cache.k_pages)
        assert torch.equal(a.cache.v_pages, b.cache.v_pages)


def test_step_without_room():
    """A sequence whose table is full, one without a page for the token and one of negative
    length: not appended; the attention is over the tokens that are there."""
    s = Server([32, 16, 5, 9], 2, 64, 16, torch.float32, fill=1.0, room=0)
    s.table_host[1, 1] = -1
    s.table.copy_(s.table_host[:, :s.table.shape[1]])
    s.lengths[2] = -1
    q, k, v = s.queries(4), s.normal(4, 2, 64), s.normal(4, 2, 64)
    kp, vp = s.cache.k_pages.clone(), s.cache.v_pages.clone()
    out = s.cache.step(q, k.cuda(), v.cuda(), s.table[:, :2], s.lengths)
    _appended(s, 3, 9, k[3:], v[3:], kp, vp)
    assert torch.equal(s.cache.k_pages, kp) and torch.equal(s.cache.v_pages, vp)
    s.k[2], s.v[2] = s.k[2][:0], s.v[2][:0]
    s.k[3], s.v[3] = torch.cat((s.k[3], k[3:])), torch.cat((s.v[3], v[3:]))
    R.check(out, *s.want(q))


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_then_steps(dtype):
    """As a server uses them: prompts rotated and appended, then decode steps with the lengths
    advanced on the device; each step against attention over the unpaged rows in 64 bits."""
    H, G, D, ps = 2, 4, 64, 16
    kw = dict(scaling="bands", factor=8.0, context=32)
    s = Server([0, 0, 0], H, D, ps, dtype, rot=D, room=80, **kw)
    counts = [37, 1, 64]
    k, v = s.normal(102, H, D), s.normal(102, H, D)
    off = torch.tensor([0, 37, 38, 102], dtype=torch.int32).cuda()
    s.cache.append(k.cuda(), v.cuda(), s.table, s.lengths, off)
    s.lengths += torch.tensor(counts, dtype=torch.int32).cuda()

    def rotated(x, first):  # keys as the pages hold them, rounded to their type
        y, tol = R.rotate(x, torch.arange(first, first + x.shape[0]), D, **kw)
        return y, tol

    rows = [rotated(k[a:b], 0) for a, b in ((0, 37), (37, 38), (38, 102))]
    s.k, s.v = [r[0] for r in rows], [v[:37], v[37:38], v[38:]]
    kerr = [r[1] for r in rows]
    for step in range(12):
        q, k1, v1 = s.queries(H * G), s.normal(3, H, D), s.normal(3, H, D)
        out = s.cache.step(q, k1.cuda(), v1.cuda(), s.table, s.lengths)
        for i in range(3):
            y, tol = rotated(k1[i:i + 1], s.k[i].shape[0])
            s.k[i], kerr[i] = torch.cat((s.k[i], y)), torch.cat((kerr[i], tol))
            s.v[i] = torch.cat((s.v[i], v1[i:i + 1]))
        s.lengths += 1
        want, tol = s.want(q)
        # the keys' roundings: scores off by scale |q| . err(k), weights by twice that
        for i in range(3):
            qa = q[i].cpu().double().abs().view(H, G, D).amax((1, 2)) * 2  # of a rotated query
            ds = (kerr[i].sum(-1).amax(0) * qa / math.sqrt(D))[:, None, None]
            va = s.v[i].double().abs().amax(0)[:, None]
            tol[i] += (2 * ds * va).expand(H, G, D).reshape(H * G, D)
        R.check(out, want, tol, f"step {step}")


# ---------------------------------------------------------------- streams and graphs

def test_captured_steps():
    """A captured step, its lengths advanced by the graph, replayed: each replay's output and
    pages are the eager ones', with eager calls on the same cache between the replays."""
    def make():
        return Server([40, 0, 130, 2047], 2, 64, 16, torch.bfloat16, rot=64, room=40, fill=0.0)

    a, b, other = make(), make(), make()
    q, k, v = a.queries(8), a.normal(4, 2, 64).cuda(), a.normal(4, 2, 64).cuda()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = a.cache.step(q, k, v, a.table, a.lengths)
        a.lengths.add_(1)
    for i in range(6):
        for x in (q, k, v):
            x.copy_(a.normal(*x.shape))
        graph.replay()
        want = b.cache.step(q, k, v, b.table, b.lengths)
        b.lengths += 1
        assert torch.equal(out, want), i
        assert torch.equal(a.cache.k_pages, b.cache.k_pages)
        # other lengths through the same workspace
        eager = a.cache.attend(q, other.table, other.lengths)
        assert eager.shape == out.shape
        torch.cuda.synchronize()


def test_two_graphs_on_one_cache():
    s = Server([3000, 500], 2, 128, 64, torch.float16)
    q1, q2 = s.queries(2), s.queries(32)
    want1, want2 = s.attend(q1), s.attend(q2, window=700)
    stream, g1, g2 = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, stream=stream):
        o1 = s.attend(q1)
    with torch.cuda.graph(g2, stream=stream):
        o2 = s.attend(q2, window=700)
    for _ in range(4):
        o1.zero_(), o2.zero_()
        g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, want1) and torch.equal(o2, want2)


def test_two_caches_at_once():
    """Handles have workspaces of their own: calls on two streams do not disturb each other."""
    a, b = (Server([20000, 9000], 2, 64, 64, torch.bfloat16, seed=i) for i in range(2))
    qa, qb = a.queries(4), b.queries(4)
    want = a.attend(qa), b.attend(qb)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            x = a.attend(qa)
        with torch.cuda.stream(s2):
            y = b.attend(qb)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


# ---------------------------------------------------------------- refusals

def test_no_sequences():
    s = Server([4], 2, 64, 16, torch.float32)
    none, no = s.table[:0], s.lengths[:0]
    q, k = torch.empty(0, 4, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda")
    assert s.cache.attend(q, none, no).shape == (0, 4, 64)
    assert s.cache.step(q, k, k, none, no).shape == (0, 4, 64)
    s.cache.append(k, k, none, no)
    s.cache.append(k, k, s.table, s.lengths, torch.zeros(2, dtype=torch.int32, device="cuda"))


def test_refusals():
    s = Server([4, 9], 2, 64, 16, torch.float16)
    c, t, n = s.cache, s.table, s.lengths
    q, k = s.queries(4), s.normal(2, 2, 64).cuda()
    off = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    for kind, call in (
            (TypeError, lambda: c.attend(q.float(), t, n)),
            (TypeError, lambda: c.attend(q, t.long(), n)),
            (TypeError, lambda: c.attend(q, t, n.long())),
            (ValueError, lambda: c.attend(q[..., :32], t, n)),
            (ValueError, lambda: c.attend(q[:1], t, n)),
            (ValueError, lambda: c.attend(q, t[:1], n)),
            (ValueError, lambda: c.attend(q, t[0], n)),
            (ValueError, lambda: c.attend(q.cpu(), t, n)),
            (ValueError, lambda: c.attend(q, t.cpu(), n)),
            (ValueError, lambda: c.attend(q, t, n, window=0)),
            (ValueError, lambda: c.attend(q, t, n, scale=0.0)),
            (RuntimeError, lambda: c.attend(q, t, n, scale=float("nan"))),
            (RuntimeError, lambda: c.attend(q[:, :3], t, n)),
            (RuntimeError, lambda: c.attend(q, t, n, out=q)),
            (RuntimeError, lambda: c.attend(q, t, n, out=q[:, :1].expand(2, 4, 64))),
            (ValueError, lambda: c.attend(q, t, n, out=q[:, :2])),
            (RuntimeError, lambda: c.attend(q, t, n, out=c.k_pages[:2, 0, :4])),
            (RuntimeError, lambda: c.append(c.k_pages[:2, 0, :2], k, t, n)),
            (ValueError, lambda: c.attend(q, s.table_host.cuda()[:, ::2], n)),
            (ValueError, lambda: c.append(k, k[:1], t, n)),
            (ValueError, lambda: c.append(k[:, :1], k[:, :1], t, n)),
            (ValueError, lambda: c.append(k[:1], k[:1], t, n)),
            (ValueError, lambda: c.append(k, k, t, n, off[:2])),
            (ValueError, lambda: c.append(k, k, t, n, off.long())),
            (ValueError, lambda: c.step(q, k[:1], k[:1], t, n)),
            (RuntimeError, lambda: c.step(q, q[:, :2], k, t, n, out=q)),
            (ValueError, lambda: PagedCache(c.k_pages, c.v_pages[:1])),
            (TypeError, lambda: PagedCache(c.k_pages.double(), c.v_pages.double())),
            (ValueError, lambda: PagedCache(c.k_pages[:, :, ::2], c.v_pages[:, :, ::2])),
            (ValueError, lambda: PagedCache(c.k_pages.cpu(), c.v_pages.cpu())),
            (RuntimeError, lambda: PagedCache(c.k_pages, c.k_pages)),
            (RuntimeError, lambda: PagedCache.allocate(2, 1, 8, 64)),
            (RuntimeError, lambda: PagedCache.allocate(2, 1, 16, 60)),
            (RuntimeError, lambda: PagedCache.allocate(2, 1, 16, 264)),
            (RuntimeError, lambda: PagedCache.allocate(2, 1, 16, 64, rotary=Rotary(128)))):
        with pytest.raises(kind):
            call()
    R.check(s.attend(q), *s.want(q))  # refused calls left nothing behind


@pytest.mark.parametrize("scale,kind", [
    (1e-60, ValueError), (-1e-46, ValueError),  # 0 in fp32, which stands for 1/sqrt(dim)
    (3e38, RuntimeError), (-3e38, RuntimeError), (1e300, (RuntimeError, TypeError))])
def test_scales_beyond_fp32(scale, kind):
    s = Server([4, 9], 2, 64, 16, torch.float16)
    q, k = s.queries(4), s.normal(2, 2, 64).cuda()
    with pytest.raises(kind):
        s.cache.attend(q, s.table, s.lengths, scale=scale)
    with pytest.raises(kind):
        s.cache.step(q, k, k, s.table, s.lengths, scale=scale)
    R.check(s.attend(q), *s.want(q))


def test_c_refusals():
    """The C entries by themselves: null pointers, counts and strides that make no sense."""
    k = torch.zeros(2, 2, 16, 64, device="cuda")
    v = torch.zeros_like(k)
    args = [k.data_ptr(), v.data_ptr(), 2, 16, 2, 64, 0, None]
    for i, x in ((0, None), (1, None), (0, k.data_ptr() + 4), (2, 0), (2, -1), (3, 0), (3, 24),
                 (3, 1 << 17), (4, 0), (4, 1 << 20), (5, 0), (5, 12), (5, 512), (6, 3),
                 (1, k.data_ptr() + 4096)):
        bad = list(args)
        bad[i] = x
        assert L.adaptq_paged_create(*bad) is None, (i, x)
        assert _lib.last_error().startswith("adaptq_paged_create: ")
    h = L.adaptq_paged_create(*args)
    assert h, _lib.last_error()
    t = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    q, o = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda")
    at = [h, q.data_ptr(), o.data_ptr(), 4, 256, 1024, 256, 1024, t.data_ptr(), 1, 1, n.data_ptr(),
          2, 0.0, 0, None]
    assert L.adaptq_paged_attend_device(*at) == 0
    for i, x in ((0, None), (1, None), (2, None), (2, q.data_ptr()), (3, 0), (3, 3), (3, -4), (4, 2),
                 (5, 2 ** 62), (6, 128), (7, 512), (8, None), (8, t.data_ptr() + 1), (9, -1), (9, 2),
                 (11, None), (12, -1), (12, 2 ** 31 - 1), (13, float("inf")), (14, -1)):
        bad = list(at)
        bad[i] = x
        assert L.adaptq_paged_attend_device(*bad) == -1, (i, x)
        assert _lib.last_error().startswith("adaptq_paged_attend_device: ")
    ap = [h, q.data_ptr(), o.data_ptr(), 2, 256, 1024, 256, 1024, t.data_ptr(), 1, 1, n.data_ptr(),
          2, None, None]
    assert L.adaptq_paged_append_device(*ap) == 0
    for i, x in ((0, None), (1, None), (2, None), (1, k.data_ptr()), (3, -1), (3, 1), (4, 6),
                 (8, None), (10, 0), (11, None), (12, 3), (13, n.data_ptr() + 2)):
        bad = list(ap)
        bad[i] = x
        assert L.adaptq_paged_append_device(*bad) == -1, (i, x)
    torch.cuda.synchronize()
    L.adaptq_paged_destroy(h)
    L.adaptq_paged_destroy(None)
    L.adaptq_rotary_destroy(None)


def test_handle_outlives_its_rotary():
    s = Server([50], 2, 64, 16, torch.float32, rot=64)
    r = L.adaptq_rotary_create(64, 0, 10000.0, 0, 1.0, 0, 0.0, 0.0, 0.0)
    h = L.adaptq_paged_create(s.cache.k_pages.data_ptr(), s.cache.v_pages.data_ptr(),
                              s.cache.pages, 16, 2, 64, 0, r)
    assert h, _lib.last_error()
    L.adaptq_rotary_destroy(r)
    junk = torch.randn(1 << 20, device="cuda")
    q = s.queries(4)
    out = torch.empty_like(q)
    assert L.adaptq_paged_attend_device(h, q.data_ptr(), out.data_ptr(), 4, 256, 1024, 256, 1024,
                                        s.table.data_ptr(), s.table.shape[1], s.table.stride(0),
                                        s.lengths.data_ptr(), 1, 0.0, 0, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, s.attend(q)) and junk is not None
    L.adaptq_paged_destroy(h)
