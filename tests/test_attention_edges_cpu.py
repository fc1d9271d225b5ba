"""Refusals of ops.attention_bwd that need no GPU."""
import pytest
import torch


def test_backward_without_the_forwards_statistics():
    """attention_fwd(want_lse=False) leaves no lse to go back with."""
    from recommendsystem_amd import ops
    from recommendsystem_amd._lib import RSError
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RSError, match="want_lse"):
        ops.attention_bwd(x, x, x, x, x, None)
    with pytest.raises(RSError, match="want_lse"):
        ops.attention_bwd(x, x, x, x, None, torch.zeros(1, 1, 2))
