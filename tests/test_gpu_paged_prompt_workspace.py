"""Which prompts take a workspace from their caller: those of few rows use the cache's own."""
import pytest
import torch

import test_gpu_paged_prompt as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def api(torch_dev):
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    P.PagedCache, P.Rotary = PagedCache, Rotary


def allocated(call):
    """Bytes that a call takes from torch beside its output."""
    call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = call()
    torch.cuda.synchronize()
    size = out.numel() * out.element_size()
    return torch.cuda.max_memory_allocated() - before - (size + 511) // 512 * 512


def test_few_rows_take_none():
    c = P.Case([16000], [4], 8, 4, 128, 64, torch.bfloat16)
    none = torch.zeros(4, dtype=torch.int32)
    cuda = none.cuda()
    assert allocated(c.run) == 0
    assert allocated(lambda: c.cache.attend(c.q, c.p.table, c.p.lengths, c.offsets, window=99)) == 0
    assert allocated(lambda: c.cache.attend(c.q, c.p.table, c.p.lengths, c.offsets, prefix=cuda)) == 0
    # the many-row kernel's, whose pieces are joined
    assert allocated(lambda: c.cache.attend(c.q, c.p.table, c.p.lengths, c.offsets, first=cuda)) > 1 << 20
    assert allocated(lambda: c.cache.attend(c.q, c.p.table, c.p.lengths, c.offsets, prefix=cuda,
                                            window=99)) > 1 << 20
    for kw in ({}, dict(first=none), dict(prefix=none), dict(window=99),
               dict(window=99, prefix=none)):
        c.check(**kw)


def test_the_c_entry_asks_for_what_it_uses():
    """A workspace is refused where it is too small and used, and not looked at where it is not."""
    import ctypes as C
    from adaptq_amd import _lib
    lib = _lib.lib
    c = P.Case([9000], [4], 2, 4, 64, 64, torch.float16)
    h = lib.adaptq_paged_create(c.p.k_pages.data_ptr(), c.p.v_pages.data_ptr(), c.p.pages, 64, 2, 64,
                                1, None)
    assert h
    out, zero = torch.empty_like(c.q), torch.zeros(4, dtype=torch.int32).cuda()
    row, table = 128, c.p.table

    def call(scores, space, size):
        return lib.adaptq_paged_prompt_device(
            h, c.q.data_ptr(), out.data_ptr(), 8, 4, row, 8 * row, row, 8 * row, table.data_ptr(),
            table.shape[1], table.stride(0), c.p.lengths.data_ptr(), 1, c.offsets.data_ptr(), 0.0,
            C.byref(scores), space, size, torch.cuda.current_stream().cuda_stream)

    def need(scores):
        return lib.adaptq_paged_prompt_scores_workspace(h, 8, 4, 1, table.shape[1],
                                                        None if scores is None else C.byref(scores))

    few = _lib.Scores(0.0, 0, None, None, None)
    many = _lib.Scores(0.0, 0, None, None, zero.data_ptr())
    most = lib.adaptq_paged_prompt_workspace(h, 8, 4, 1, table.shape[1])
    assert need(few) == need(None) == 0 and need(many) == most > 0
    assert call(few, None, 0) == 0
    first = out.clone()
    assert call(many, None, 0) == -1 and b"workspace" in lib.adaptq_last_error()
    space = torch.empty(most, dtype=torch.uint8, device="cuda")
    assert call(many, space.data_ptr(), most - 1) == -1
    assert call(many, space.data_ptr(), most) == 0
    P.R.check(first, *c.want())
    P.R.check(out, *c.want())
    torch.cuda.synchronize()
    lib.adaptq_paged_destroy(h)
