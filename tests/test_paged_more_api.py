"""The entries of masked attention, eviction and 4-bit pages without a GPU: what they refuse
before any device call is made."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from adaptq_amd import _lib
    return _lib.lib


def test_paged4_create_rejects(lib):
    page = 0x1000000
    good = [page, 2 * page, 4, 16, 2, 64, 0, None]
    for i, x in ((0, None), (1, None), (6, 3), (6, -1), (2, 0), (4, 0), (4, 40000), (3, 0), (3, 8),
                 (3, 40), (3, 1 << 17), (5, 0), (5, 40), (5, 72), (5, 288), (0, page + 8), (1, page),
                 (1, page + 4 * 2 * 16 * 34 - 16)):
        args = list(good)
        args[i] = x
        assert lib.adaptq_paged4_create(*args) is None, (i, x)
        assert lib.adaptq_last_error().startswith(b"adaptq_paged4_create: ")
        assert b"HIP" not in lib.adaptq_last_error()


def test_null_handles(lib):
    lib.adaptq_paged4_destroy(None)
    seqs = (None, 1, 1, None, 1)
    rows = (None, None, 1, 0, 0, 0, 0)
    for name, args in (
            ("adaptq_paged_prompt_device", (None, None, 1, 1, 0, 0, 0, 0, *seqs, None, 0.0, None, None,
                                            0, None)),
            ("adaptq_paged_attend_scores_device", (None, None, 1, 0, 0, 0, 0, *seqs, 0.0, None, None, 0,
                                                   0, None, 0, None)),
            ("adaptq_paged_step_scores_device", (None, None, 0, 0, 0, 0, None, None, 1, 0, 0, 0, 0,
                                                 *seqs, 0.0, None, None, 0, 0, None, 0, None)),
            ("adaptq_paged_evict_device", (None, 0, 0, *seqs, 1, 0, None, 0, 0, None, None)),
            ("adaptq_paged4_append_device", (*rows, *seqs, None, None)),
            ("adaptq_paged4_read_device", (None, None, 1, *seqs, None, None)),
            ("adaptq_paged4_attend_device", (None, None, 1, 0, 0, 0, 0, *seqs, 0.0, None, None)),
            ("adaptq_paged4_step_device", (None, None, 0, 0, 0, 0, None, None, 1, 0, 0, 0, 0, *seqs,
                                           0.0, None, None))):
        assert getattr(lib, name)(None, *args) == -1
        assert lib.adaptq_last_error() == name.encode() + b": null handle"
    assert lib.adaptq_paged_prompt_workspace(None, 4, 4, 4, 4) == 0
    assert lib.adaptq_paged_weights_workspace(None, 4, 4, 4) == 0


def test_python_side_rejects_the_cpu():
    import torch
    from adaptq_amd.paged import PagedCache4
    pool = torch.zeros(2, 1, 16, 34, dtype=torch.uint8)
    with pytest.raises(ValueError):
        PagedCache4(pool, pool.clone())
    with pytest.raises(TypeError):
        PagedCache4(pool.float(), pool.float())
    with pytest.raises(ValueError):
        PagedCache4(pool[..., :30], pool[..., :30])
    with pytest.raises(ValueError):
        PagedCache4.allocate(2, 1, 16, 40)
