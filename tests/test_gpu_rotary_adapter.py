"""AdaptQAttention with a rotary on the types that the module takes without one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [("float64", "float64", "float64"),
                                   ("float16", "float32", "bfloat16"),
                                   ("float32", "float32", "float16")])
def test_other_and_mixed_types(torch_dev, types):
    """They go through fp32, as without a rotary: the same outputs as fp32 rows rotated before."""
    from adaptq_amd.rotary import Rotary
    from adaptq_amd.torch_adapter import AdaptQAttention
    H, D = 3, 64
    rotary = Rotary(D)
    a, b = AdaptQAttention(D, H, seed=3, rotary=rotary), AdaptQAttention(D, H, seed=3)
    g = torch.Generator().manual_seed(1)
    for t in range(4):
        q, k, v = (torch.randn(1, H, D, generator=g).to(getattr(torch, x)).cuda() for x in types)
        pos = torch.tensor([t], dtype=torch.int32).cuda()
        rq, rk = rotary(pos, q.float(), k.float())
        y = a(q, k, v)
        assert y.dtype == q.dtype and torch.equal(y, b(rq, rk, v.float()).to(q.dtype))
