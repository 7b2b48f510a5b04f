"""Tables and batches past what the embedding kernels count, on the CPU: the entry point refuses before it launches anything."""
import pytest
import torch

from system_lab_b200.ops import cuda, lookup


def test_tables_past_the_limit_take_the_oracle():
    """Slices of the table are counted in 32 bits: at 2^31 - 1 rows their number passes them."""
    row = torch.zeros(1, 8)
    assert lookup.supports(row.expand(2 ** 30, 8), torch.float32)
    for rows in (2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31):
        assert not lookup.supports(row.expand(rows, 8), torch.float32)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the entry point is called without memory")
@pytest.mark.parametrize("rows,vocab", [(4, 2 ** 31 - 1), (4, 2 ** 30 + 1), (2 ** 30 + 1, 4), (4, 0), (0, 4)])
def test_entry_point_refuses(rows, vocab):
    try:
        fn = cuda.lib().slab_embedding_bwd
    except Exception as e:
        pytest.skip(f"kernel library not built: {e}")
    assert fn(None, None, 0, None, 0, None, None, rows, 8, vocab, 8, 1.0, 0, None) == -10
