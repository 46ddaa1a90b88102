"""What the Python calls of the 8-bit linear path do besides launching: errors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def test_out_of_memory_is_torchs_error():
    """An output that no GPU has room for (8 TB): torch.OutOfMemoryError, which callers catch to take a smaller batch,
    and the next call works."""
    import bbh

    n = 2_000_000
    q, s = torch.zeros(n, 16, dtype=torch.int8, device=DEV), torch.ones(n, device=DEV)
    with pytest.raises(torch.OutOfMemoryError, match="out of memory"):
        bbh.linear_i8(q, s, q, s)
    assert bool((bbh.linear_i8(q[:5], s[:5], q[:7], s[:7]) == 0).all())
