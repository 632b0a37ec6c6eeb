"""The rotary and paged-cache entries of the C ABI without a GPU: what they refuse before
any device call is made."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from adaptq_amd import _lib
    return _lib.lib


GOOD = dict(rotary_dim=64, interleaved=0, base=10000.0, scaling=0, factor=1.0, context=0,
            slow=0.0, fast=0.0, amplitude=0.0)


@pytest.mark.parametrize("bad", [
    dict(rotary_dim=0), dict(rotary_dim=-2), dict(rotary_dim=63), dict(rotary_dim=1026),
    dict(scaling=-1), dict(scaling=5), dict(base=1.0), dict(base=float("nan")),
    dict(base=float("inf")), dict(factor=0.5), dict(factor=float("inf")), dict(amplitude=-1.0),
    dict(amplitude=float("nan")), dict(scaling=2, rotary_dim=2), dict(scaling=3),
    dict(scaling=4, context=-1), dict(scaling=4, context=64, slow=4.0, fast=4.0),
    dict(scaling=3, context=64, slow=-1.0), dict(scaling=3, context=64, fast=float("nan")),
])
def test_rotary_create_rejects(lib, bad):
    assert lib.adaptq_rotary_create(*{**GOOD, **bad}.values()) is None
    assert lib.adaptq_last_error().startswith(b"adaptq_rotary_create: ")
    assert b"HIP" not in lib.adaptq_last_error()


def test_paged_create_rejects(lib):
    page = 0x1000000
    good = [page, 2 * page, 4, 16, 2, 64, 0, None]
    for i, x in ((0, None), (1, None), (6, 3), (6, -1), (2, 0), (4, 0), (4, 40000), (3, 0), (3, 8),
                 (3, 40), (3, 1 << 17), (5, 0), (5, 60), (5, 264), (0, page + 8), (1, page)):
        args = list(good)
        args[i] = x
        assert lib.adaptq_paged_create(*args) is None, (i, x)
        assert lib.adaptq_last_error().startswith(b"adaptq_paged_create: ")
        assert b"HIP" not in lib.adaptq_last_error()


def test_null_handles(lib):
    lib.adaptq_rotary_destroy(None)
    lib.adaptq_paged_destroy(None)
    assert lib.adaptq_rotary_device(None, None, 1, 64, 0, None, 0, 1, 1, 0, None) == -1
    assert lib.adaptq_last_error() == b"adaptq_rotary_device: null handle"
    assert lib.adaptq_paged_append_device(None, None, None, 1, 0, 0, 0, 0, None, 1, 1, None, 1, None,
                                          None) == -1
    assert lib.adaptq_last_error() == b"adaptq_paged_append_device: null handle"
    assert lib.adaptq_paged_attend_device(None, None, None, 1, 0, 0, 0, 0, None, 1, 1, None, 1, 0.0,
                                          0, None) == -1
    assert lib.adaptq_last_error() == b"adaptq_paged_attend_device: null handle"
    assert lib.adaptq_paged_step_device(None, None, None, 0, 0, 0, 0, None, None, 1, 0, 0, 0, 0, None,
                                        1, 1, None, 1, 0.0, 0, None) == -1
    assert lib.adaptq_last_error() == b"adaptq_paged_step_device: null handle"


def test_python_side_rejects_the_cpu():
    import torch
    from adaptq_amd.paged import PagedCache
    from adaptq_amd.rotary import Rotary
    with pytest.raises(ValueError):
        Rotary(64, device="cpu")
    with pytest.raises(ValueError):
        Rotary(64, scaling="none")
    x = torch.zeros(2, 2, 16, 64)
    with pytest.raises(ValueError):
        PagedCache(x, torch.zeros_like(x))
    with pytest.raises(TypeError):
        PagedCache(x.double(), x.double())


@pytest.mark.parametrize("amplitude", [1e39, 1e300])
def test_rotary_create_rejects_an_amplitude_beyond_fp32(lib, amplitude):
    """It would be infinite on the device, and 0 times it NaN."""
    assert lib.adaptq_rotary_create(*{**GOOD, "amplitude": amplitude}.values()) is None
    assert b"amplitude" in lib.adaptq_last_error() and b"HIP" not in lib.adaptq_last_error()
