"""Refusals of the packed-sequence calls that need no device."""
import pytest
import torch

from r97training_b200 import _lib as L
from r97training_b200 import ops


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu"), "meta"])
def test_rope_tables_of_another_kind_of_device(device):
    """Not tables on the current GPU in place of those asked for."""
    with pytest.raises(L.R97bError):
        ops.rope_tables(8, 64, 1e4, device=device)
