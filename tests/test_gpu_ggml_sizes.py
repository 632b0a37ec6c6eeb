"""A ggml append of more values than a launch has threads."""
import ctypes as C

import numpy as np
import pytest
import torch

from adaptq_amd import _lib

pytestmark = pytest.mark.gpu
L = _lib.lib


def test_append_of_more_than_2_32_values(torch_dev):
    """2^22 + 64 tokens of 8 heads of 128, one row for all of them (34 GB of copies): the ring of
    64 holds what 64 such tokens leave."""
    H, D, cap, n = 8, 128, 64, 2 ** 22 + 64
    g = torch.Generator().manual_seed(0)
    k, v, q = (torch.randn(H, D, generator=g).cuda() for _ in range(3))
    outs = []
    for tokens in (cap, n):
        m = L.adaptq_mha_create(H, D, 4, 4, cap, 7, 0.0, 0)
        assert m, _lib.last_error()
        assert L.adaptq_ggml_append_f32_device(
            m, C.c_void_p(k.data_ptr()), C.c_void_p(v.data_ptr()), D, H, tokens, D * 4, 0, D * 4, 0,
            0, None) == 0, _lib.last_error()
        out = torch.empty(H, D, device="cuda")
        assert L.adaptq_ggml_attn_f32_device(m, C.c_void_p(q.data_ptr()), D, H, 1, D * 4, H * D * 4,
                                             C.c_void_p(out.data_ptr()), D * 4, H * D * 4,
                                             None) == cap, _lib.last_error()
        torch.cuda.synchronize()
        outs.append(out.cpu().numpy())
        L.adaptq_mha_destroy(m)
    assert np.isfinite(outs[0]).all() and np.array_equal(outs[0], outs[1])
