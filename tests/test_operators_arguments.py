# SPDX-License-Identifier: MIT OR Apache-2.0
"""Arguments that the operators refuse, on the CPU (before a device is looked at)."""

import pytest
import torch

import candle_fused_attn as cfa


@pytest.mark.parametrize("shape", [(3, 4), (3, 1), (2, 3), (5,), (1,), (1, 2, 4), ()])
def test_positions_of_other_shapes(shape):
    x, f = torch.zeros(2, 3, 4, 8), torch.ones(4, dtype=torch.float64)
    at = torch.zeros(shape, dtype=torch.int64)
    for call in (lambda: cfa.rotary(x, at, f), lambda: cfa.rotary_qkv(torch.zeros(2, 4, 72), 3, at, f)):
        with pytest.raises(cfa.FusedAttentionError, match=r"positions \[4\], \[2, 4\] or \[2, 1\] expected"):
            call()


@pytest.mark.parametrize("shape", [(4,), (2, 4), (1, 4), (2, 1)])
def test_positions_that_are_taken(shape):
    """One a token, or a sequence's one for all of its tokens."""
    x, f = torch.zeros(2, 3, 4, 8), torch.ones(4, dtype=torch.float64)
    with pytest.raises(cfa.FusedAttentionError, match="CUDA tensors required"):
        cfa.rotary(x, torch.zeros(shape, dtype=torch.int32), f)
