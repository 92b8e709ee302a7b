"""Calls that tree_attention refuses before anything is launched."""
import math

import pytest
import torch


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, math.nan, math.inf, 1e-50, 1e300])
def test_refuses_a_scale_that_is_not_above_0(scale):
    """(0 and below would be 1 / sqrt(D) in the kernels.)"""
    from torchplusplus_amd.attention import tree_attention
    q, c = torch.zeros(1, 1, 2, 64, dtype=torch.float16), torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="softmax_scale"):
        tree_attention(q, c, c, torch.zeros(1, dtype=torch.int32), softmax_scale=scale)
