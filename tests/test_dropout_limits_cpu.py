"""The limits of the dropout's rate."""
import pytest
import torch

from system_lab_b200 import ops


def test_rates_up_to_the_limit():
    """The rate is taken to the nearest multiple of 2^-16: from 1 - 2^-17 on that is one, and everything would be dropped."""
    x = torch.randn(4, 8)
    ops.dropout(x, 1 - 2.0 ** -16, 1)
    ops.dropout(x, 1 - 2.0 ** -17 - 2.0 ** -40, 1)
    for p in (1 - 2.0 ** -17, 1 - 2.0 ** -18):
        with pytest.raises(ValueError, match="below 1 - 2\\^-17"):
            ops.dropout(x, p, 1)
