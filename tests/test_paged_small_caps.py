"""Caps that fp32 does not hold: 0 means none to the library, so a cap that rounds to it would be
left out without an error (on the CPU: the check is made before any call)."""
import pytest
import torch


@pytest.mark.parametrize("cap", [5e-324, 1e-60, 1e-46, 1e-40, 7e-31, 0.0, -1.0, -1e-60,
                                 float("nan"), -float("inf")])
def test_refused(cap):
    from adaptq_amd.paged import PagedCache, PagedCache4
    for kind in (PagedCache, PagedCache4):
        cache = kind.__new__(kind)
        cache.device = torch.device("cpu")
        with pytest.raises(ValueError, match="softcap"):
            cache._scores(1, 4, cap, None, None, None)


@pytest.mark.parametrize("cap", [2.0 ** -100, 1e-6, 30.0, 1e38])
def test_taken(cap):
    from adaptq_amd.paged import PagedCache
    cache = PagedCache.__new__(PagedCache)
    cache.device = torch.device("cpu")
    assert cache._scores(1, 4, cap, None, None, None) == (cap, 0, 0, 0)
