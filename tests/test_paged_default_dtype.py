"""What the paged caches allocate is of the type that the library writes, whatever torch's default
type is (on the CPU, over a handle that takes the addresses and writes nothing)."""
import pytest
import torch


@pytest.fixture
def default(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


@pytest.mark.parametrize("default", [torch.float16, torch.bfloat16, torch.float64], indirect=True)
@pytest.mark.parametrize("tokens,sequences", [(3, 3), (3, 0), (0, 0)])
def test_rows_that_are_read_back(default, tokens, sequences):
    from adaptq_amd.paged import PagedCache4

    class Handle:
        calls = 0

        def read(self, *args):
            self.calls += 1

    cache = PagedCache4.__new__(PagedCache4)
    cache.device, cache.heads, cache.dim = torch.device("cpu"), 2, 64
    cache._handle = Handle()
    cache._stream = lambda: 0
    table = torch.zeros(sequences, 1, dtype=torch.int32)
    lengths = torch.zeros(sequences, dtype=torch.int32)
    offsets = torch.zeros(sequences + 1, dtype=torch.int32)
    for x in cache.read(tokens, table, lengths, offsets):
        assert x.dtype == torch.float32 and x.shape == (tokens, 2, 64)
    assert cache._handle.calls == (tokens > 0 and sequences > 0)
